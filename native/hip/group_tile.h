// The tiled kernels of the grouped products: a BM x BN output tile per workgroup, WM x WN waves, operand panels
// of 128 bytes along the reduction (64 elements of 16 bits, or 128 of fp8, one scale block) staged through LDS.
#pragma once

#include "group_common.h"

template <int DT_, int SC_, bool ATR_, bool BTR_, int BM_, int BN_, int WM_, int WN_, int NBUF_>
struct TileCfg {
  static constexpr int DT = DT_, SC = SC_, BM = BM_, BN = BN_, WM = WM_, WN = WN_;
  static constexpr bool ATR = ATR_, BTR = BTR_;
  static constexpr int ES = DT == kFp8 ? 1 : 2;          // bytes an element
  static constexpr int PB = 128, NBUF = NBUF_;            // bytes a panel is wide; panels in the ring
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
};

// Byte of 16-byte chunk q of row r in a K-major panel: rows of 128 bytes, chunks permuted by the row so that
// the fragment reads (16 rows, one chunk) spread over the banks.
__device__ __forceinline__ int km_swizzle(int r) { return r & 7; }
__device__ __forceinline__ int km_at(int r, int q) { return r * 128 + ((q ^ km_swizzle(r)) << 4); }

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
  } else if (from < upto && upto >= N) {                  // the row's last 16 bytes, moved down: one load
    unsigned __int128 last;
    __builtin_memcpy(&last, row + (size_t)(upto - N) * ES, 16);
    v = __builtin_bit_cast(gi4, last >> ((from + N - upto) * (8 * ES)));
  } else if (from < upto) {
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
    return lds_chunk(base + blk0 * 16 * C::PB + km_at(j16, s * 4 + g) + blk * 16 * C::PB);
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
  const gi4 x = lds_chunk(base + blk0 * 2048 + km_at(j16, g) + blk * 2048);
  const gi4 y = lds_chunk(base + blk0 * 2048 + km_at(j16, g + 4) + blk * 2048);
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

// A tile: what it reads and where it writes.
struct TileWork {
  TileOperands t;
  char* c;
  int rows, cols;
};

// The launch's work items, one for each tile -- except that the tiles past the last whole round of the `slots`
// workgroups that run at once, which would keep few of them busy for a whole tile's time, are cut into 2 or 4 parts by
// rows, as many as still fit one round.
template <class C>
struct TilePlan {
  RowTiles rows;
  const int* by_size = nullptr;                            // weight gradients: GroupsBySize in LDS, where they have been saved
  int tiles_m, tiles_n, whole, over, parts, items;

  TilePlan() = default;
  __device__ __forceinline__ explicit TilePlan(const GroupArgs& g) {
    tiles_n = (g.cols + C::BN - 1) / C::BN;
    if constexpr (C::ATR) {                                // weight gradients: whole tiles of every expert
      tiles_m = (g.rows + C::BM - 1) / C::BM;
      items = tiles_m * tiles_n * g.experts;
    } else {
      rows.init(g, g.rows, C::BM);
      tiles_m = rows.tiles;
      over = g.slots > 0 ? tiles_m * tiles_n % g.slots : 0;
      whole = tiles_m * tiles_n - over;
      parts = over == 0 ? 1 : 4 * over <= g.slots ? 4 : 2 * over <= g.slots ? 2 : 1;
      items = whole + over * parts;
    }
  }

  // Of one wave.
  static constexpr int kWords = RowTiles::kWords + 6;
  static_assert(RowTiles::kWords >= GroupsBySize::kWords, "either in the same place");
  __device__ __forceinline__ void save(const GroupArgs& g, int* at) const {
    if constexpr (C::ATR) {
      if (GroupsBySize::sorted(g)) GroupsBySize(g, g.red).save(g, at);
    } else {
      if (rows.off != nullptr) rows.save(at);
    }
    at += RowTiles::kWords;
    at[0] = tiles_m;
    at[1] = tiles_n;
    at[2] = items;
    if constexpr (!C::ATR) {
      at[3] = whole;
      at[4] = over;
      at[5] = parts;
    }
  }
  __device__ __forceinline__ void load(const GroupArgs& g, const int* at) {
    if constexpr (C::ATR) by_size = at;
    else rows.load(g, g.rows, C::BM, at);
    at += RowTiles::kWords;
    tiles_m = __builtin_amdgcn_readfirstlane(at[0]);
    tiles_n = __builtin_amdgcn_readfirstlane(at[1]);
    items = __builtin_amdgcn_readfirstlane(at[2]);
    if constexpr (!C::ATR) {
      whole = __builtin_amdgcn_readfirstlane(at[3]);
      over = __builtin_amdgcn_readfirstlane(at[4]);
      parts = __builtin_amdgcn_readfirstlane(at[5]);
    }
  }

  // item < items; false: a part without rows
  __device__ __forceinline__ bool work(const GroupArgs& g, int item, TileWork& w) {
    TileOperands& t = w.t;
    int tm, tn;
    t.lda_b = g.lda * C::ES;
    t.ldb_b = g.ldb * C::ES;
    if constexpr (C::ATR) {
      // an expert's tiles over all XCDs: whole experts to an XCD would leave those with the short ones idle
      const int per = tiles_m * tiles_n, place = item / per;
      int e = place, begin = 0, end = g.red;
      tile_coords(xcd_remap(item - place * per, per), tiles_m, tiles_n, tm, tn);
      if (!GroupsBySize::sorted(g)) {
        if (g.offsets) group_rows(g.offsets, e, g.red, begin, end);
      } else if (by_size != nullptr) {
        e = __builtin_amdgcn_readfirstlane(by_size[place]);
        begin = __builtin_amdgcn_readfirstlane(by_size[64 + place]);
        end = __builtin_amdgcn_readfirstlane(by_size[128 + place]);
      } else {
        const GroupsBySize groups(g, g.red);
        e = __builtin_ctzll(__ballot((int)(threadIdx.x & 63) < g.experts && groups.rank == place));
        begin = __builtin_amdgcn_readlane(groups.begin, e);
        end = __builtin_amdgcn_readlane(groups.end, e);
      }
      t.a = (const char*)g.a + (size_t)begin * g.lda * C::ES;
      t.b = (const char*)g.b + (size_t)begin * g.ldb * C::ES;
      t.a_col0 = tm * C::BM;
      t.b_col0 = tn * C::BN;
      t.a_cols = g.rows;
      t.b_cols = g.cols;
      t.red = end - begin;
      w.rows = min(C::BM, g.rows - tm * C::BM);
      w.cols = min(C::BN, g.cols - tn * C::BN);
      w.c = (char*)g.c + 2 * ((size_t)e * g.c_expert + (size_t)tm * C::BM * g.ldc + (size_t)tn * C::BN);
      return true;
    } else {
      int tile, part = 0;
      if (item < whole) {
        tile = xcd_remap(item, whole);
      } else {
        const int at = xcd_remap(item - whole, over * parts);
        tile = whole + at / parts;
        part = at % parts;
      }
      tile_coords(tile, tiles_m, tiles_n, tm, tn);
      RowTile rt = rows.find(tm);
      if (parts > 1 && item >= whole) {
        rt.row0 += part * (C::BM / parts);
        rt.row_end = min(rt.row_end, rt.row0 + C::BM / parts);
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
      w.rows = t.a_rows;
      w.cols = t.b_rows;
      w.c = (char*)g.c + 2 * ((size_t)rt.row0 * g.ldc + (size_t)tn * C::BN);
      return true;
    }
  }
};

// The result through LDS, which the loop has left: whole rows of the tile at a time, 16 bytes a lane (straight from
// the accumulators a store would write 32 bytes of each of 16 rows). Accumulator [i][j] of a lane holds row
// 16 (i WM + wm) + (lane & 15), columns 16 j + 4 (lane >> 4) + 0..3 of the wave's part: B is the matrix instruction's
// first operand, so a lane's four values lie along a row. 16-byte chunk c of row r lies at c ^ (r & 15): neither side
// conflicts. Rows that start with a line of 128 bytes are streamed past the caches. Others share their lines with another
// workgroup's: those go the ordinary way, so that the L2 writes whole lines (32 experts' 1032 x 2056 weight gradients of 65
// rows each take 1.8 times as long streamed).
template <class C>
__device__ __forceinline__ void tile_store_rows(const GroupArgs& g, char* lds, char* c_tile, int c_rows, int c_cols, int wm, int wn,
                                                const gf4 (&acc)[C::NI][C::NJ]) {
  static_assert(C::BM * C::BN * 2 <= C::LDS, "the tile fits the ring");
  constexpr int OUT = C::DT == kFp16 ? kFp16 : kBf16;
  const bool lines = (((uintptr_t)g.c | (uintptr_t)(g.ldc * 2) | (uintptr_t)(g.c_expert * 2)) & 127) == 0;
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
      if (lines) store_c16(at, v);
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

// One operand's panels by LDS-DMA (buffer_load ... lds): a wave instruction (a piece) fills 1 KiB of LDS in lane
// order, so the permutation of the chunks goes on the addresses that the lanes read. A wave's pieces are STEP panel rows
// apart, a multiple of the permutations' period, so a lane's offset is that of its first piece and the rest is the same
// for all lanes. Panel rows at or past `limit`, and lanes with nothing to read, ask for kNowhere: zeros, whatever lies
// there. Panel rows are the operand's rows (K-major) or reduction steps (reduction-major).
template <class C, bool TR, int ROWS>
struct PanelDma {
  static constexpr int WAVES = C::THREADS / 64;
  static constexpr int PIECES = ROWS * C::PB / 1024 / WAVES;
  static constexpr int LANES = TR ? ROWS / 8 : C::PB / 16;          // lanes, and chunks, of a panel row
  static constexpr int STEP = WAVES * 64 / LANES, ALL = TR ? C::KT : ROWS;
  static_assert(PIECES * WAVES * 1024 == ROWS * C::PB, "whole pieces");
  static_assert(STEP % 16 == 0, "the permutations' period");
  unsigned off;
  int row;                                                          // of the lane's first piece

  // the 16-byte chunk of its row that the lane reads
  __device__ __forceinline__ int chunk(int lane) const {
    const int q = lane % LANES;
    if constexpr (TR) return (((q >> 1) ^ rm_swizzle(row)) << 1) | (q & 1);
    else return q ^ km_swizzle(row);
  }
  __device__ __forceinline__ void init(int wave, int lane, unsigned ld, int col0, int cols) {
    row = wave * (64 / LANES) + lane / LANES;
    const int q = chunk(lane);
    if constexpr (TR) off = col0 + q * 8 < cols ? (unsigned)row * ld + (unsigned)(col0 + q * 8) * 2 : kNowhere;
    else off = (unsigned)row * ld + q * 16;
  }
  // K-major, the last panel: `left` reduction steps of it exist
  __device__ __forceinline__ void cut(int lane, int left) {
    if constexpr (!TR) off = chunk(lane) * 16 < left * C::ES ? off : kNowhere;
  }
  __device__ __forceinline__ void load(char* lds, const char* panel, int wave, unsigned ld, int limit) const {
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)panel, 0, 0x7fffffff, 0x00020000);
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const unsigned o = limit >= ALL || row + i * STEP < limit ? off : kNowhere;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (g_lds_ptr)(lds + (i * WAVES + wave) * 1024), 16, o, i * STEP * ld, 0, 0);
    }
  }
};

// The scales of a panel by LDS-DMA: waves 0 .. BM / 64 - 1 fetch a row's each lane, the next wave the columns', the
// others nothing.
template <class C>
__device__ __forceinline__ void scale_lanes(const GroupArgs& g, const TileOperands& t, int wave, int lane, unsigned& soff,
                                            const char*& base, long long& step) {
  constexpr int SB = C::SC == kScaleF32 ? 4 : 1;
  // (both operands' values first: a choice between the structs' members would put the structs into memory)
  const bool of_a = wave < C::BM / 64, of_b = wave == C::BM / 64;
  const int r = of_a ? wave * 64 + lane : lane, n = of_a ? t.a_rows : of_b ? min((t.b_rows + kScaleBlock - 1) / kScaleBlock, C::BN / kScaleBlock) : 0;
  const unsigned ar = (unsigned)(g.as_row * SB), br = (unsigned)(g.bs_row * SB);
  const long long ak = g.as_k * SB, bk = g.bs_k * SB;
  const char *as = t.as, *bs = t.bs;
  soff = r < n ? (unsigned)r * (of_a ? ar : br) : kNowhere;
  base = of_a ? as : bs;
  step = of_a ? ak : bk;
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
  long long step_s;
  unsigned soff, lda, ldb;
  int wave, lane, nk, left, a_rows, b_rows;

  __device__ __forceinline__ TileLoader(const GroupArgs& g, const TileOperands& t, int wave_, int lane_)
      : pa(t.a), pb(t.b), ps(t.as), step_s(0), soff(kNowhere), lda((unsigned)t.lda_b), ldb((unsigned)t.ldb_b), wave(wave_),
        lane(lane_), a_rows(t.a_rows), b_rows(t.b_rows) {
    nk = (t.red + C::KT - 1) / C::KT;
    left = t.red - (nk - 1) * C::KT;
    da.init(wave, lane, lda, t.a_col0, t.a_cols);
    db.init(wave, lane, ldb, t.b_col0, t.b_cols);
    if constexpr (C::SC != kScaleNone) scale_lanes<C>(g, t, wave, lane, soff, ps, step_s);
  }
  // panel kt (the next one) into `base`
  __device__ __forceinline__ void issue(int kt, char* base) {
    const int steps = kt == nk - 1 ? left : C::KT;
    if (steps < C::KT) {
      da.cut(lane, left);
      db.cut(lane, left);
    }
    da.load(base, pa, wave, lda, C::ATR ? steps : a_rows);
    db.load(base + C::OPA, pb, wave, ldb, C::BTR ? steps : b_rows);
    if constexpr (C::SC != kScaleNone) {
      scale_load<C>(base + C::OPA + C::OPB, ps, wave, soff);
      ps += step_s;
    }
    pa += C::ATR ? (size_t)C::KT * lda : C::PB;
    pb += C::BTR ? (size_t)C::KT * ldb : C::PB;
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

// A workgroup a tile, its panels in a ring of NBUF, NBUF - 1 of them in flight. At panel t a counted wait
// retires t's pieces only, a bare s_barrier publishes them, and panel t + NBUF - 1 goes into the buffer that
// every wave left at t - 1.
//
// Bound by what a CU's panels bring in from the L2, 40 to 50 KB a microsecond (a 128 x 128 tile reads 32 KB for 2 * 128^3
// fp8 operations), or for few rows a group by the weights: fp8 128 x 4096 x 4096 13.5 us, 512 x 8192 x 8192 52.9 (1300
// TFLOP/s); bf16 16 groups of 32 rows, 2048 x 4096, 56 us (4.8 TB/s of weights), of 128 rows, 2048 x 2048, 41.
template <class C>
__global__ void __launch_bounds__(C::THREADS) __attribute__((amdgpu_waves_per_eu(C::EU, C::EU)))
group_tile_dma(const GroupArgs g) {
  __shared__ __attribute__((aligned(16))) char lds[C::LDS];     // the only LDS object: see tile_step
  if (rest_block(g, C::THREADS)) return;
  TilePlan<C> plan(g);
  TileWork w;
  if ((int)blockIdx.x >= plan.items || !plan.work(g, blockIdx.x, w)) return;
  const int c_rows = w.rows, lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / C::WN, wn = wave % C::WN;
  TileLoader<C> ld(g, w.t, wave, lane);
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
  tile_store_rows<C>(g, lds, w.c, c_rows, w.cols, wm, wn, acc);
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
  // where they are in a stage: every read is a lane's address and a 16-bit constant
  static constexpr int B = 0, LO = C::OPB, HI = LO + HALF, STAGE = HI + HALF;
  // a half tile's panels: a ring of three, the last of them over the results
  static constexpr int HSTAGE = HI;
  static constexpr int OUT = 2 * STAGE, OUT_END = 3 * HSTAGE > OUT + 8 * 2048 ? 3 * HSTAGE : OUT + 8 * 2048;
  static constexpr int SCALES = OUT_END, PLAN = SCALES + 4 * C::SCB, LDS = PLAN + 1024, STORES = 2 * C::NI;
  static_assert(LDS <= 160 * 1024 && (RowTiles::kWords + 6) * 4 <= 1024, "one CU's LDS");
  using DmaA = PanelDma<C, C::ATR, HM>;
  using DmaB = PanelDma<C, C::BTR, C::BN>;
  static constexpr int P1 = DmaA::PIECES + DmaB::PIECES + (C::SC != kScaleNone ? 1 : 0), P2 = DmaA::PIECES;
  static_assert(C::WM == 2 && C::WN == 4 && C::NBUF == 2, "two groups of four waves, two panels");
};

// A value that is the same in all lanes, as the compiler should know: it stays in scalar registers.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ size_t uniform(size_t v) {
  return (size_t)(unsigned)uniform((int)(v >> 32)) << 32 | (unsigned)uniform((int)v);
}
__device__ __forceinline__ const char* uniform(const char* p) { return (const char*)uniform((size_t)p); }

template <class C>
struct PingPongLoader {
  using P = PingPong<C>;
  typename P::DmaA lo, hi;                       // (K-major, they differ in the rows that exist alone)
  typename P::DmaB b;
  const char *pa, *pb, *ps;
  long long step_s;
  unsigned soff, lda, ldb;
  int wave, lane, nk, left, a_rows, b_rows;

  __device__ __forceinline__ PingPongLoader(const GroupArgs& g, const TileOperands& t, int wave_, int lane_)
      : pa(uniform(t.a)), pb(uniform(t.b)), ps(t.as), step_s(0), soff(kNowhere), lda((unsigned)uniform((int)t.lda_b)),
        ldb((unsigned)uniform((int)t.ldb_b)), wave(wave_), lane(lane_), a_rows(uniform(t.a_rows)), b_rows(uniform(t.b_rows)) {
    const int red = uniform(t.red);
    nk = (red + C::KT - 1) / C::KT;
    left = red - (nk - 1) * C::KT;
    lo.init(wave, lane, lda, t.a_col0, t.a_cols);
    if constexpr (C::ATR) hi.init(wave, lane, lda, t.a_col0 + P::HM, t.a_cols);
    b.init(wave, lane, ldb, t.b_col0, t.b_cols);
    if constexpr (C::SC != kScaleNone) {
      scale_lanes<C>(g, t, wave, lane, soff, ps, step_s);
      ps = uniform(ps);
      step_s = (long long)uniform((size_t)step_s);
    }
  }
  __device__ __forceinline__ const char* a_panel(int kt) const { return pa + (size_t)kt * (C::ATR ? (size_t)C::KT * lda : C::PB); }
  // B, A's upper half and the scales of panel kt into the stage at `base`
  __device__ __forceinline__ void issue_lo(int kt, char* base, char* ring) {
    const int steps = kt == nk - 1 ? left : C::KT;
    typename P::DmaA a = lo;
    if (steps < C::KT) {
      a.cut(lane, left);
      b.cut(lane, left);
    }
    b.load(base + P::B, pb + (size_t)kt * (C::BTR ? (size_t)C::KT * ldb : C::PB), wave, ldb, C::BTR ? steps : b_rows);
    a.load(base + P::LO, a_panel(kt), wave, lda, C::ATR ? steps : a_rows);
    if constexpr (C::SC != kScaleNone) scale_load<C>(ring + (kt & 3) * C::SCB, ps + kt * step_s, wave, soff);
  }
  __device__ __forceinline__ void issue_hi(int kt, char* base) {
    const int steps = kt == nk - 1 ? left : C::KT;
    typename P::DmaA a = C::ATR ? hi : lo;
    if (steps < C::KT) a.cut(lane, left);
    const char* panel = a_panel(kt);
    if constexpr (!C::ATR) panel += (size_t)P::HM * lda;
    a.load(base + P::HI, panel, wave, lda, C::ATR ? steps : a_rows - P::HM);
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

// A tile's first panels, into stages that no wave reads any more.
template <class C>
__device__ __forceinline__ void pp_prologue(char* lds, PingPongLoader<C>& ld, int rows) {
  using P = PingPong<C>;
  if (ld.nk == 0) return;
  const bool half = rows <= C::BM / 2;
  ld.issue_lo(0, lds, lds + P::SCALES);
  if (!half) ld.issue_hi(0, lds);
  if (ld.nk > 1) ld.issue_lo(1, lds + (half ? P::HSTAGE : P::STAGE), lds + P::SCALES);
}

// wait_vm<N>, or with `stores` that many of this wave's stores (kStores) more
template <class C, int N>
__device__ __forceinline__ void pp_wait(bool stores) {
  if (stores) wait_vm<N + PingPong<C>::STORES>();
  else wait_vm<N>();
}

// After pp_prologue. `stores`: exactly PingPong::STORES of this wave's stores have been issued since, and may go on.
template <class C>
__device__ __forceinline__ void pp_loop(char* lds, PingPongLoader<C>& ld, int wave, int wm, int wn, bool stores,
                                        gf4 (&acc)[C::NI][C::NJ]) {
  using P = PingPong<C>;
  const int nk = ld.nk;
  if (nk == 0) return;
  char* const ring = lds + P::SCALES;
  if (nk > 1) pp_wait<C, P::P1 + P::P2>(stores);
  else pp_wait<C, P::P2>(stores);
  bar();
  if (wave >= 4) bar();
  for (int kt = 0; kt < nk; ++kt) {
    char* const here = lds + (kt & 1) * P::STAGE;
    char* const there = lds + (~kt & 1) * P::STAGE;
    const bool st = stores && kt == 0;
    PingPongFrags<C> f;
    pp_read_lo<C>(there, (lds_in)here, (lds_in)ring, ld, kt, wm, wn, f);
    if (kt + 1 < nk) pp_wait<C, P::P1 + P::P2>(st);       // this wave's pieces of the lower half have landed
    else wait_vm<0>();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    bar();
    __builtin_amdgcn_s_setprio(1);
    pp_mul<C, 0, P::NH>(f, acc);
    __builtin_amdgcn_s_setprio(0);
    bar();
    // (the stage's upper half, B and scales have been read by both groups: panel kt + 2's go there)
    pp_read_hi<C>(here, (lds_in)here, ring, ld, kt, wm, wn, f);
    if (kt + 2 < nk) pp_wait<C, P::P1 + P::P2>(st);       // and of the next panel's first part
    else pp_wait<C, P::P2>(st);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    bar();
    __builtin_amdgcn_s_setprio(1);
    pp_mul<C, P::NH, P::NH>(f, acc);
    __builtin_amdgcn_s_setprio(0);
    bar();
  }
  if (wave < 4) bar();
}

// A tile of at most half the rows: its upper half alone, NA of a wave's blocks. The two groups take turns here too, with
// two intervals a panel and a ring of three: panel t + 2 goes where panel t - 1 was, which both groups have read.
template <class C, int NA>
__device__ __forceinline__ void pp_half_read(char* __restrict__ into, const __attribute__((address_space(3))) char* __restrict__ from,
                                             char* ring, PingPongLoader<C>& ld, int kt, int wm, int wn, PingPongFrags<C>& f) {
  pp_frags_lo<C, NA>(from, wm, wn, f);
  pp_scales<C, NA, 0>((lds_in)ring, kt, wm, wn, f);
  if (kt + 2 < ld.nk) ld.issue_lo(kt + 2, into, ring);
}

template <class C, int NA>
__device__ __forceinline__ void pp_half_loop(char* lds, PingPongLoader<C>& ld, int wave, int wm, int wn, bool stores,
                                             gf4 (&acc)[C::NI][C::NJ]) {
  using P = PingPong<C>;
  const int nk = ld.nk;
  if (nk == 0) return;
  if (nk > 1) pp_wait<C, P::P1>(stores);
  else pp_wait<C, 0>(stores);
  bar();
  if (wave >= 4) bar();
  int buf = 0;
  for (int kt = 0; kt < nk; ++kt) {
    const bool st = stores && kt == 0;
    PingPongFrags<C> f;
    pp_half_read<C, NA>(lds + (buf == 0 ? 2 : buf - 1) * P::HSTAGE, (lds_in)lds + buf * P::HSTAGE, lds + P::SCALES, ld, kt, wm, wn, f);
    if (kt + 2 < nk) pp_wait<C, P::P1>(st);                // this wave's pieces of the next panel have landed
    else pp_wait<C, 0>(st);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    bar();
    __builtin_amdgcn_s_setprio(1);
    pp_mul<C, 0, NA>(f, acc);
    __builtin_amdgcn_s_setprio(0);
    bar();
    buf = buf == 2 ? 0 : buf + 1;
  }
  if (wave < 4) bar();
}

// The lane, as a value made here: what is computed from it stays inside the loop over the tiles (hoisted out of it, the
// addresses of a tile's start and end fill the registers that the sums need).
__device__ __forceinline__ int lane_here() {
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));
  return lane;
}

// The result while the next tile's first panels land: a wave's 16-row blocks one after the other through 2 KiB of its
// own (no barrier), 8 rows of 128 bytes a store. True: exactly STORES stores (lanes without a row or column store past
// the buffer's end, nowhere); else as many as it takes.
template <class C>
__device__ __forceinline__ bool pp_store(const GroupArgs& g, char* stage, const TileWork& w, int wm, int wn,
                                         const gf4 (&acc)[C::NI][C::NJ]) {
  constexpr int OUT = C::DT == kFp16 ? kFp16 : kBf16;
  const int lane = lane_here(), l16 = lane & 15, q = lane >> 4;
  const size_t apart = (uintptr_t)g.c | (uintptr_t)(g.ldc * 2) | (uintptr_t)(g.c_expert * 2);
  const bool fast = ((apart & 15) | (w.cols & 7)) == 0, lines = (apart & 127) == 0;
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(w.c, 0, 0x7fffffff, 0x00020000);
  const int r8 = lane >> 3, c8 = lane & 7, col = wn * C::TN + c8 * 8;
  static_assert(C::TN == 64, "a wave's rows are 128 bytes");
#pragma unroll
  for (int i = 0; i < C::NI; ++i) {
#pragma unroll
    for (int j = 0; j < C::NJ; ++j) {
      unsigned short v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = to_out<OUT>(acc[i][j][e]);
      const int c = 2 * j + (q >> 1);
      *(uint2*)(stage + l16 * 128 + ((c ^ (l16 >> 1)) << 4) + (q & 1) * 8) = make_uint2(v[0] | (unsigned)v[1] << 16, v[2] | (unsigned)v[3] << 16);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int rl = r8 + 8 * h, r = (i * C::WM + wm) * 16 + rl;
      const gi4 v = *(const gi4*)(stage + rl * 128 + ((c8 ^ (rl >> 1)) << 4));
      if (fast) {
        const unsigned at = r < w.rows && col < w.cols ? (unsigned)r * (unsigned)(g.ldc * 2) + (unsigned)col * 2 : kNowhere;
        if (lines) __builtin_amdgcn_raw_buffer_store_b128(v, rs, at, 0, 2);        // 2: streaming, as store_c16
        else __builtin_amdgcn_raw_buffer_store_b128(v, rs, at, 0, 0);
      } else if (r < w.rows) {
        unsigned short* at = (unsigned short*)w.c + (size_t)r * g.ldc + col;
        if (col + 8 <= w.cols) {
          __builtin_memcpy(at, &v, 16);
        } else {
          const unsigned short* from = (const unsigned short*)(stage + rl * 128 + ((c8 ^ (rl >> 1)) << 4));
#pragma unroll 1
          for (int e = 0; col + e < w.cols; ++e) at[e] = from[e];
        }
      }
    }
  }
  return fast;
}

// The launch's arguments, read here: kept in scalar registers from the start they would not leave the loops enough.
__device__ __forceinline__ GroupArgs args_here() {
  const __attribute__((address_space(4))) char* at = (const __attribute__((address_space(4))) char*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(at));
  GroupArgs g;
  __builtin_memcpy(&g, (const char*)at, sizeof(g));
  return g;
}

// The workgroup's next item with work: workgroup b of `slots` takes one of every round of `slots` items. Inside a
// round it keeps its XCD (b & 7) and moves on by 5 places, or the same workgroups would get all of the short tiles that
// come every 8 items. A weight gradient's items come in order of their length: there every other round runs backwards (16
// experts of 40 to 1500 rows, 2056 x 1032: 68.9 -> 65.0 us).
template <class C>
__device__ __forceinline__ bool pp_next(const GroupArgs& g, TilePlan<C>& plan, int& round, TileWork& w) {
  const int b = blockIdx.x;
  for (;; ++round) {
    const long long base = (long long)round * g.slots;
    if (base >= plan.items) return false;
    int place = b;
    if constexpr (C::ATR) place = (round & 1) != 0 ? g.slots - 1 - b : b;
    else if ((g.slots & 7) == 0) place = ((b >> 3) + 5 * round) % (g.slots >> 3) * 8 + (b & 7);
    if (base + place < plan.items && plan.work(g, (int)base + place, w)) {
      ++round;
      return true;
    }
  }
}

// One workgroup a CU, for all of the launch's tiles: the next tile's first panels are fetched before the result of the
// last one is stored, so that the stores, and the wait for the first panels, run under each other and under the next
// tile's loop (a workgroup a tile: 11 us a tile between the loops, 9.4 for fp8; like this 6 and 8). What the tiles'
// starts and ends need is kept in LDS and read there, not in registers across the loops.
//
// Bound by the matrix unit, which the card clocks down under it: 8192^3 fp8 444 to 504 us by card (2180 to 2480 TFLOP/s; 539
// as the median of 30 from a cold start; each further 4096 of K at 2620, e8m0 2970), bf16 of 8192 x 8192 x 4096 361 us (1520; 1630).
// With groups, by their last tiles: 8 of 2048 rows on average, 8192 x 4096 bf16, 815 to 877 us (1350 to 1250; 913 from a cold
// start), 26 fp8 ones of 590, 4096 x 4096, 315 to 330 (1640).
template <class C>
__global__ void __launch_bounds__(C::THREADS) __attribute__((amdgpu_waves_per_eu(2, 2))) group_tile_pp(const GroupArgs args) {
  using P = PingPong<C>;
  __shared__ __attribute__((aligned(16))) char lds[P::LDS];     // the only LDS object: see tile_step
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / C::WN, wn = wave % C::WN;
  int* const kept = (int*)(lds + P::PLAN);
  TileWork w;
  int round = 0;
  bool more;
  {
    TilePlan<C> plan(args);
    more = pp_next<C>(args, plan, round, w);
    if (wave == 0) plan.save(args, kept);
  }
  __syncthreads();
  if (more) {
    PingPongLoader<C> ld(args, w.t, wave, lane);
    pp_prologue<C>(lds, ld, w.rows);
    int stores = 0;
    while (more) {
      gf4 acc[C::NI][C::NJ];
#pragma unroll
      for (int i = 0; i < C::NI; ++i)
#pragma unroll
        for (int j = 0; j < C::NJ; ++j) acc[i][j] = gf4{0.f, 0.f, 0.f, 0.f};
      if (w.rows > C::BM / 2) pp_loop<C>(lds, ld, wave, wm, wn, stores, acc);
      else if (w.rows > C::BM / 4) pp_half_loop<C, P::NH>(lds, ld, wave, wm, wn, stores, acc);
      else pp_half_loop<C, P::NH / 2>(lds, ld, wave, wm, wn, stores, acc);
      const GroupArgs g = args_here();
      TileWork next;
      TilePlan<C> plan;
      plan.load(g, kept);
      more = uniform((int)pp_next<C>(g, plan, round, next));
      if (more) {
        ld = PingPongLoader<C>(g, next.t, wave, lane_here());
        pp_prologue<C>(lds, ld, next.rows);
      }
      stores = uniform((int)pp_store<C>(g, lds + P::OUT + wave * 2048, w, wm, wn, acc));
      w.c = (char*)uniform((const char*)next.c);
      w.rows = uniform(next.rows);
      w.cols = uniform(next.cols);
    }
  }
  const GroupArgs g = args_here();
  zero_rest_rows(g, blockIdx.x, g.slots, C::THREADS);
}
