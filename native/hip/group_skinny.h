// The forward product for few rows a group (decode steps): bound by reading the weights once.
//
// A workgroup owns MT x 16 rows of one group and NJ x 16 columns; its KW waves take the reduction's 128-byte panels
// in turn (panel w, w + KW, ..), so the workgroup streams KW x 128 consecutive bytes of every weight row at a
// time. Weights go from memory straight to the matrix instructions' operand registers, a batch of U panels in flight
// while the one before is multiplied; nothing is shared between waves until the end, so there is no barrier and
// no LDS in the loop. Rows of the operand that do not exist are loads past the buffer's end: they cost no
// traffic. Batches of one panel: 16 rows of 8192 x 8192 fp8 take 17.3 us, with batches of two 18.4, of four 20.6; 64 experts of
// 4096 x 2048 fp8 with a row each 93.7, 101.5, 144.9 (and 94.8 as a loop over panels without batches: the compiler then orders
// the waits otherwise). The waves' partial sums are joined through LDS in wave order: the same bits every time.
//
// 16 rows of 8192 x 8192 fp8: 17.3 us one after the other over the same weights (3.9 TB/s of weights; a large copy reads and
// writes 5.1), 20.3 over other weights each time, and 18.2 to 20.8 in a trace; 64 rows over 64 experts of 4096 x 2048 fp8, 37 of
// them busy: 51 to 56 us (5.9 TB/s); 8 rows over 6 busy experts of 4096 x 4096 bf16: 33 us (6.0 TB/s).
#pragma once

#include "group_tile.h"

template <int DT_, int SC_, int MT_, int NJ_, int KW_, int ALIGN_ = 16>
struct SkinnyCfg {
  static constexpr int ALIGN = ALIGN_;           // 16: rows of whole, aligned 16-byte chunks; 4, 1: rows that start on so many bytes
  static constexpr int DT = DT_, SC = SC_, MT = MT_, NJ = NJ_, KW = KW_;
  static constexpr int U = 1;                    // panels of a batch, see above
  static constexpr int ES = DT == kFp8 ? 1 : 2;
  static constexpr int ROWS = 16 * MT, COLS = 16 * NJ, THREADS = 64 * KW;
  static constexpr int LDS = KW * ROWS * COLS * 4;
  static_assert(kScaleBlock % COLS == 0, "one column scale a tile");
};

// A panel's operands in registers: two 16-byte chunks (g and g + 4 of the row's 8) for each 16 rows or columns.
template <class C>
struct SkinnyPanel {
  gi4 a[C::MT][2], b[C::NJ][2];
  int sa[C::MT], sb;
};

// The same of rows that start anywhere: the words that hold the chunks (`moved`: not yet moved down).
template <class C>
struct SkinnyWords {
  Any16 a[C::MT][2], b[C::NJ][2];
  int sa[C::MT], sb;
  bool moved;
};

template <class C>
__device__ __forceinline__ void skinny_panel(const SkinnyWords<C>& w, const unsigned (&shift_a)[C::MT], const unsigned (&shift_b)[C::NJ],
                                             SkinnyPanel<C>& p) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int m = 0; m < C::MT; ++m) p.a[m][h] = any16_get(w.a[m][h], w.moved ? shift_a[m] : 0);
#pragma unroll
    for (int j = 0; j < C::NJ; ++j) p.b[j][h] = any16_get(w.b[j][h], w.moved ? shift_b[j] : 0);
  }
#pragma unroll
  for (int m = 0; m < C::MT; ++m) p.sa[m] = w.sa[m];
  p.sb = w.sb;
}

// Panel k of rows without whole aligned chunks.
template <class C>
__device__ __forceinline__ void skinny_load(SkinnyPanel<C>& p, const char* const (&pa)[C::MT], const char* const (&pb)[C::NJ], int k,
                                            int q0, int red) {
  const unsigned at = (unsigned)k * 128u;
  const bool whole = at + 128u <= (unsigned)red * C::ES;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const unsigned from = at + (unsigned)(q0 + 4 * h) * 16u;
    if (whole) {
#pragma unroll
      for (int m = 0; m < C::MT; ++m) __builtin_memcpy(&p.a[m][h], pa[m] + from, 16);
#pragma unroll
      for (int j = 0; j < C::NJ; ++j) __builtin_memcpy(&p.b[j][h], pb[j] + from, 16);
    } else {                                           // the last panel, or none
#pragma unroll
      for (int m = 0; m < C::MT; ++m) p.a[m][h] = load_chunk<C::ES>(pa[m], (int)(from / C::ES), red);
#pragma unroll
      for (int j = 0; j < C::NJ; ++j) p.b[j][h] = load_chunk<C::ES>(pb[j], (int)(from / C::ES), red);
    }
  }
}

template <class C>
__device__ __forceinline__ void skinny_load(SkinnyWords<C>& p, const char* const (&pa)[C::MT], const char* const (&pb)[C::NJ], int k,
                                            int q0, int red) {
  const unsigned at = (unsigned)k * 128u;
  p.moved = at + 128u <= (unsigned)red * C::ES;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const unsigned from = at + (unsigned)(q0 + 4 * h) * 16u;
    if (p.moved) {
#pragma unroll
      for (int m = 0; m < C::MT; ++m) any16_load(p.a[m][h], pa[m] + from);
#pragma unroll
      for (int j = 0; j < C::NJ; ++j) any16_load(p.b[j][h], pb[j] + from);
    } else {                                           // the last panel, or none
#pragma unroll
      for (int m = 0; m < C::MT; ++m) p.a[m][h] = Any16{load_chunk<C::ES>(pa[m], (int)(from / C::ES), red), 0};
#pragma unroll
      for (int j = 0; j < C::NJ; ++j) p.b[j][h] = Any16{load_chunk<C::ES>(pb[j], (int)(from / C::ES), red), 0};
    }
  }
}

__device__ __forceinline__ gi4 buffer_chunk(__amdgpu_buffer_rsrc_t rs, unsigned off) {
  return __builtin_bit_cast(gi4, __builtin_amdgcn_raw_buffer_load_b128(rs, off, 0, 0));
}

template <int SC>
__device__ __forceinline__ int buffer_scale(__amdgpu_buffer_rsrc_t rs, unsigned off) {
  if constexpr (SC == kScaleF32) return (int)__builtin_amdgcn_raw_buffer_load_b32(rs, off, 0, 0);
  else return (int)__builtin_amdgcn_raw_buffer_load_b8(rs, off, 0, 0);
}

template <class C>
__device__ __forceinline__ void skinny_mul(const SkinnyPanel<C>& p, gf4 (&acc)[C::MT][C::NJ]) {
#pragma unroll
  for (int m = 0; m < C::MT; ++m) {
    if constexpr (C::DT == kFp8) {
      const gi8 av = __builtin_shufflevector(p.a[m][0], p.a[m][1], 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
      for (int j = 0; j < C::NJ; ++j) {
        const gi8 bv = __builtin_shufflevector(p.b[j][0], p.b[j][1], 0, 1, 2, 3, 4, 5, 6, 7);
        if constexpr (C::SC == kScaleF32) {
          const float s = __builtin_bit_cast(float, p.sa[m]) * __builtin_bit_cast(float, p.sb);
          const gf4 d = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(bv, av, gf4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
#pragma unroll
          for (int q = 0; q < 4; ++q) acc[m][j][q] = fmaf(d[q], s, acc[m][j][q]);
        } else {
          acc[m][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(bv, av, acc[m][j], 0, 0, 0, p.sb, 0, p.sa[m]);
        }
      }
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < C::NJ; ++j) {
          if constexpr (C::DT == kFp16)
            acc[m][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(gh8, p.b[j][h]),
                                                                __builtin_bit_cast(gh8, p.a[m][h]), acc[m][j], 0, 0, 0);
          else
            acc[m][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(gbf8, p.b[j][h]),
                                                                 __builtin_bit_cast(gbf8, p.a[m][h]), acc[m][j], 0, 0, 0);
        }
    }
  }
}

template <class C, int ALIGN>
struct SkinnyLoaded { using T = SkinnyPanel<C>; };
template <class C>
struct SkinnyLoaded<C, 1> { using T = SkinnyWords<C>; };

template <class C>
__global__ void __launch_bounds__(C::THREADS) group_skinny(const GroupArgs g) {
  __shared__ __attribute__((aligned(16))) char lds[C::LDS];
  if (rest_block(g, C::THREADS)) return;
  const int tiles_n = (g.cols + C::COLS - 1) / C::COLS;
  const int tm = blockIdx.x / tiles_n, n0 = (blockIdx.x - tm * tiles_n) * C::COLS;
  RowTiles row_tiles;
  row_tiles.init(g, g.rows, C::ROWS);
  if (tm >= row_tiles.tiles) return;
  const RowTile rt = row_tiles.find(tm);
  const int lane = threadIdx.x & 63, l16 = lane & 15, q0 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rows = min(C::ROWS, rt.row_end - rt.row0), cols = min(C::COLS, g.cols - n0);
  constexpr int S = C::SC == kScaleF32 ? 4 : 1;
  const auto rsrc = [](const void* p) { return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, 0x7fffffff, 0x00020000); };
  const __amdgpu_buffer_rsrc_t ra = rsrc((const char*)g.a + (size_t)rt.row0 * g.lda * C::ES);
  const __amdgpu_buffer_rsrc_t rb = rsrc((const char*)g.b + ((size_t)rt.expert * g.b_expert + (size_t)n0 * g.ldb) * C::ES);
  __amdgpu_buffer_rsrc_t rsa = ra, rsb = rb;
  if constexpr (C::SC != kScaleNone) {
    rsa = rsrc((const char*)g.a_scale + (size_t)rt.row0 * g.as_row * S);
    rsb = rsrc((const char*)g.b_scale + ((size_t)rt.expert * g.bs_expert + (size_t)(n0 / kScaleBlock) * g.bs_row) * S);
  }
  unsigned oa[C::MT], ob[C::NJ], osa[C::MT];
#pragma unroll
  for (int m = 0; m < C::MT; ++m) {
    const int r = m * 16 + l16;
    oa[m] = r < rows ? (unsigned)r * (unsigned)(g.lda * C::ES) + q0 * 16 : kNowhere;
    osa[m] = r < rows ? (unsigned)r * (unsigned)(g.as_row * S) : kNowhere;
  }
#pragma unroll
  for (int j = 0; j < C::NJ; ++j) {
    const int c = j * 16 + l16;
    ob[j] = c < cols ? (unsigned)c * (unsigned)(g.ldb * C::ES) + q0 * 16 : kNowhere;
  }
  const unsigned bytes = (unsigned)g.red * C::ES;
  const unsigned as_k = (unsigned)(g.as_k * S), bs_k = (unsigned)(g.bs_k * S);
  const int nk = (g.red + 128 / C::ES - 1) / (128 / C::ES);
  // Operands without whole aligned chunks: a lane's rows and columns by their address, the last existing one in place of one
  // that does not exist (it multiplies into results that are not stored).
  const char *pa[C::MT], *pb[C::NJ];
  unsigned shift_a[C::MT], shift_b[C::NJ];
  if constexpr (C::ALIGN < 16) {
#pragma unroll
    for (int m = 0; m < C::MT; ++m) {
      pa[m] = (const char*)g.a + (size_t)(rt.row0 + min(m * 16 + l16, rows - 1)) * g.lda * C::ES;
      shift_a[m] = (unsigned)(uintptr_t)pa[m] & 3;
    }
#pragma unroll
    for (int j = 0; j < C::NJ; ++j) {
      pb[j] = (const char*)g.b + ((size_t)rt.expert * g.b_expert + (size_t)(n0 + min(j * 16 + l16, cols - 1)) * g.ldb) * C::ES;
      shift_b[j] = (unsigned)(uintptr_t)pb[j] & 3;
    }
  }
  // panel k: `at` is added to offsets that may already be past the end; they stay there (both under 2^31)
  using Loaded = typename SkinnyLoaded<C, C::ALIGN>::T;
  const auto load = [&](Loaded& p, int k) {
    const unsigned at = (unsigned)k * 128u;
    if constexpr (C::ALIGN < 16) {
      skinny_load<C>(p, pa, pb, k, q0, g.red);
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bool in = at + (unsigned)(q0 + 4 * h) * 16u < bytes;
#pragma unroll
        for (int m = 0; m < C::MT; ++m) p.a[m][h] = buffer_chunk(ra, in ? oa[m] + at + h * 64u : kNowhere);
#pragma unroll
        for (int j = 0; j < C::NJ; ++j) p.b[j][h] = buffer_chunk(rb, in ? ob[j] + at + h * 64u : kNowhere);
      }
    }
    if constexpr (C::SC != kScaleNone) {
#pragma unroll
      for (int m = 0; m < C::MT; ++m) p.sa[m] = buffer_scale<C::SC>(rsa, k < nk ? osa[m] + (unsigned)k * as_k : kNowhere);
      p.sb = buffer_scale<C::SC>(rsb, k < nk ? (unsigned)k * bs_k : kNowhere);
    }
  };
  gf4 acc[C::MT][C::NJ];
#pragma unroll
  for (int m = 0; m < C::MT; ++m)
#pragma unroll
    for (int j = 0; j < C::NJ; ++j) acc[m][j] = gf4{0.f, 0.f, 0.f, 0.f};
  Loaded cur[C::U], nxt[C::U];
#pragma unroll
  for (int u = 0; u < C::U; ++u) load(cur[u], wave + u * C::KW);
  for (int k = wave; k < nk; k += C::U * C::KW) {
#pragma unroll
    for (int u = 0; u < C::U; ++u) load(nxt[u], k + (C::U + u) * C::KW);
#pragma unroll
    for (int u = 0; u < C::U; ++u) {
      if constexpr (C::ALIGN > 1) {
        skinny_mul<C>(cur[u], acc);
      } else {
        SkinnyPanel<C> p;
        skinny_panel<C>(cur[u], shift_a, shift_b, p);
        skinny_mul<C>(p, acc);
      }
    }
#pragma unroll
    for (int u = 0; u < C::U; ++u) cur[u] = nxt[u];
  }
  // the waves' sums through LDS: [wave][row][column]
  float* part = (float*)lds;
#pragma unroll
  for (int m = 0; m < C::MT; ++m)
#pragma unroll
    for (int j = 0; j < C::NJ; ++j)
      *(gf4*)(part + ((size_t)wave * C::ROWS + m * 16 + l16) * C::COLS + j * 16 + q0 * 4) = acc[m][j];
  __syncthreads();
  constexpr int OUT = C::DT == kFp16 ? kFp16 : kBf16;
  const bool wide = ((uintptr_t)g.c & 7) == 0 && (g.ldc & 3) == 0;
  for (int i = threadIdx.x; i < C::ROWS * C::COLS / 4; i += C::THREADS) {
    const int r = i / (C::COLS / 4), c = i % (C::COLS / 4) * 4;
    if (r >= rows) break;
    gf4 s = *(const gf4*)(part + r * C::COLS + c);
#pragma unroll
    for (int w = 1; w < C::KW; ++w) s += *(const gf4*)(part + (w * C::ROWS + r) * C::COLS + c);
    unsigned short* out = (unsigned short*)g.c + (size_t)(rt.row0 + r) * g.ldc + n0 + c;
    unsigned short v[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = to_out<OUT>(s[q]);
    if (wide && c + 4 <= cols) {
      *(uint2*)out = make_uint2(v[0] | (unsigned)v[1] << 16, v[2] | (unsigned)v[3] << 16);
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (c + q < cols) out[q] = v[q];
    }
  }
}
