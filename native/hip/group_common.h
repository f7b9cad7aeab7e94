// Shared pieces of the grouped and block-scaled matrix products (gemm_group.hip).
//
//   C[r, c] = sum_k A(r, k) B(c, k)
//
// in one of three modes over rows sorted by expert (expert e owns the rows offsets[e] .. offsets[e + 1]):
//
//   forward  C[t, n] = sum_k a[t, k] bt[e(t), n, k]          ragged rows, both operands K-major
//   dgrad    C[t, k] = sum_n dc[t, n] bt[e(t), n, k]         ragged rows, B stored reduction-major
//   wgrad    C[e, n, k] = sum_{t of e} dc[t, n] a[t, k]      ragged reduction, both reduction-major
//
// "K-major": the reduction index is the contiguous one; "reduction-major": it is the row index. A product
// without experts is a forward one whose single group owns every row (offsets == nullptr).
// Operands are bf16 / fp16 (16 bits, no scales) or fp8 e4m3 with one scale per row (A) or per 128 columns
// (B) and 128 reduction steps. The sums are held in float32.
#pragma once

#include "gemm_tile_common.h"

enum : int { kModeForward = 0, kModeDgrad = 1, kModeWgrad = 2 };
enum : int { kBf16 = 0, kFp16 = 1, kFp8 = 2 };
enum : int { kScaleNone = 0, kScaleF32 = 1, kScaleE8 = 2 };

constexpr int kScaleBlock = 128;

// Mirrored field by field by ops/_lib.py. Leading dimensions and strides in elements.
struct GroupArgs {
  const void* a;
  const void* b;
  void* c;
  const void* a_scale;
  const void* b_scale;
  const int* offsets;                        // experts + 1 device ints, or null: one group of all rows
  long long lda, ldb, ldc, b_expert, c_expert;
  long long as_row, as_k, bs_expert, bs_row, bs_k;
  int rows, cols, red, experts;              // ragged extent: `rows` (forward, dgrad) or `red` (wgrad)
  int mode, dtype, scale, zero_rest;         // zero_rest: rows that no expert owns are written as zeros
  int padded;                                // rows are readable to their next multiple of 16 bytes
  int slots;                                 // workgroups that run at once; set by the dispatch
};

namespace {

typedef int gi4 __attribute__((ext_vector_type(4)));
typedef int gi8 __attribute__((ext_vector_type(8)));
typedef int gi2 __attribute__((ext_vector_type(2)));
typedef float gf4 __attribute__((ext_vector_type(4)));
typedef __bf16 gbf8 __attribute__((ext_vector_type(8)));
typedef _Float16 gh8 __attribute__((ext_vector_type(8)));
typedef short gs4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) gs4* gs4_lds;

// The rows [begin, end) of expert e. The offsets live on the device and are not checked by the host, so
// they are clamped here: whatever they hold, no row outside the operands is touched.
__device__ __forceinline__ void group_rows(const int* __restrict__ off, int e, int total, int& begin, int& end) {
  begin = min(max(off[e], 0), total);
  end = min(max(off[e + 1], begin), total);
}

// The row tile `t` of the ragged rows, counted over the experts' tiles of `bm` rows in order; false past the
// last one. Every wave runs it redundantly over registers (64 experts a step), so no barrier is needed.
struct RowTile {
  int expert, row0, row_end;
};

__device__ __forceinline__ int wave_inclusive_sum(int v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int up = __shfl_up(v, d);
    v += lane >= d ? up : 0;
  }
  return v;
}

__device__ __forceinline__ int group_tile_count(const GroupArgs& g, int total, int bm) {
  if (g.offsets == nullptr) return (total + bm - 1) / bm;
  int n = 0;
  for (int e = threadIdx.x & 63; e < g.experts; e += 64) {
    int b, x;
    group_rows(g.offsets, e, total, b, x);
    n += (x - b + bm - 1) / bm;
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) n += __shfl_xor(n, d);
  return __builtin_amdgcn_readfirstlane(n);
}

__device__ __forceinline__ bool group_find_tile(const GroupArgs& g, int total, int bm, int t, RowTile& out) {
  if (g.offsets == nullptr) {
    out = RowTile{0, t * bm, total};
    return t * (long long)bm < total;
  }
  int base = 0;
  for (int e0 = 0; e0 < g.experts; e0 += 64) {
    const int e = e0 + (threadIdx.x & 63);
    int b = 0, x = 0;
    if (e < g.experts) group_rows(g.offsets, e, total, b, x);
    const int mine = (x - b + bm - 1) / bm;
    const int upto = wave_inclusive_sum(mine);
    const unsigned long long past = __ballot(base + upto > t);
    if (past != 0) {
      const int lane = __builtin_ctzll(past);
      const int first = base + __shfl(upto, lane) - __shfl(mine, lane);
      out.expert = __builtin_amdgcn_readfirstlane(e0 + lane);
      out.row0 = __builtin_amdgcn_readfirstlane(__shfl(b, lane) + (t - first) * bm);
      out.row_end = __builtin_amdgcn_readfirstlane(__shfl(x, lane));
      return true;
    }
    base += __shfl(upto, 63);
  }
  return false;
}

// The expert with the `want`-th most rows (ties in order), up to 64 experts; above that the experts in order. A
// weight gradient's tiles take as long as their expert has rows: started with the longest, the last ones to end are
// short.
__device__ __forceinline__ int group_by_size(const GroupArgs& g, int total, int want) {
  if (g.offsets == nullptr || g.experts > 64) return want;
  const int lane = threadIdx.x & 63;
  int b = 0, x = -1;
  if (lane < g.experts) group_rows(g.offsets, lane, total, b, x);
  const int n = x - b;                               // -1 in lanes without an expert
  int rank = 0;
  for (int e = 0; e < g.experts; ++e) {
    const int other = __builtin_amdgcn_readlane(n, e);
    rank += other > n || (other == n && e < lane) ? 1 : 0;
  }
  return __builtin_ctzll(__ballot(lane < g.experts && rank == want));
}

// Most row tiles that `experts` groups of `total` rows together can have: every busy expert adds at most one
// that is not full. The host sizes the grid with it, since the offsets live on the device.
__host__ inline long long group_tile_bound(long long total, int experts, bool grouped, int bm) {
  if (!grouped) return (total + bm - 1) / bm;
  const long long busy = experts < total ? experts : total;
  return (total - busy) / bm + busy;
}

// The 16-bit value nearest to a float32 sum: the only rounding between the operands and the result.
template <int DT>
__device__ __forceinline__ unsigned short to_out(float v) {
  if constexpr (DT == kFp16) return __builtin_bit_cast(unsigned short, (_Float16)v);
  else return __builtin_bit_cast(unsigned short, (__bf16)v);
}

// Rows that no expert owns, as zeros: the whole grid walks them, each block whole rows.
__device__ __forceinline__ void zero_rest_rows(const GroupArgs& g, int cols, int block, int blocks, int threads) {
  if (!g.zero_rest || g.offsets == nullptr) return;
  const int first = min(max(g.offsets[0], 0), g.rows), last = min(max(g.offsets[g.experts], 0), g.rows);
  unsigned short* c = (unsigned short*)g.c;
  const int rest = first + (g.rows - max(last, first));
  for (int i = block; i < rest; i += blocks) {
    const int r = i < first ? i : max(last, first) + (i - first);
    unsigned short* row = c + (size_t)r * g.ldc;
    for (int j = threadIdx.x; j < cols; j += threads) row[j] = 0;
  }
}

}  // namespace
