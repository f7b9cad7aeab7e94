// fp8 e4m3 operands of the block-scaled products: one scale for each block of 128 columns of one row
// (activations) or of 128 rows (weights).
//
//   amax = max |x| over the block's finite values, at least 448 * 2^-126
//   float32 scale   s = amax / 448                              q = e4m3(x * 448 / amax)
//   e8m0 scale      s = the least 2^e with amax <= 448 * 2^e    q = e4m3(x / s)
//
// e4m3() rounds the exact quotient to the nearest value, ties to even; 448 is e4m3's largest, so nothing
// saturates. An infinity or NaN becomes NaN (e4m3 has no infinity) and leaves its block's scale alone.
//
// The quotient with a float32 scale is x times 448 / amax nearly, within 4 units in the last place. That can only change
// the e4m3 value where the exact quotient is a border between two of them, or that close to one. A border has 5
// significant bits, B. Of 16-bit inputs x = X 2^i and amax = A 2^j have at most 11: 448 x / amax is the border B 2^k where 7 X
// and B A agree but for a power of two, both integers under 2^16; so it is a border, or at least 2^-16 of it away. There the
// quotient rounded to 20 bits decides right: it moves by 2^-20 at most, and onto the border where that is
// exact (many are: half of all blocks hold an x of 3/4 or 3/8 amax). Of float32 inputs the rare values within 8 units of
// a border are compared with it exactly, in float64.
//
// Bound by the memory: 2 (4) bytes read and 1 written for each element. 16384 x 8192 bf16, a scale a row's block: 69 us (5.8
// TB/s; a large copy 5.1), 70 to 75 as one call among others; 12200 x 8256 fp32, 128 x 128 blocks: 95 us (5.3 TB/s).
#include "gemm_tile_common.h"
#include "memory_reach.h"

enum : int { kInBf16 = 0, kInFp16 = 1, kInFp32 = 2 };

struct QuantArgs {
  const void* x;
  unsigned char* q;
  void* s;
  long long ld, batch_stride;      // elements
  int batches, rows, cols;
  int dtype, block_rows, e8;
};

namespace {

typedef unsigned int qu2 __attribute__((ext_vector_type(2)));
typedef unsigned short qs2 __attribute__((ext_vector_type(2)));

constexpr int QT = 256;                // threads

// 8 consecutive elements as loaded
template <int DT>
struct Raw8 {
  static constexpr int W = DT == kInFp32 ? 8 : 4;
  unsigned int w[W];
};

template <int DT>
__device__ __forceinline__ float raw_get(const Raw8<DT>& r, int i) {
  if constexpr (DT == kInFp32) return __builtin_bit_cast(float, r.w[i]);
  const unsigned int h = (r.w[i >> 1] >> ((i & 1) * 16)) & 0xffff;
  if constexpr (DT == kInBf16) return __builtin_bit_cast(float, h << 16);
  return (float)__builtin_bit_cast(_Float16, (unsigned short)h);
}

// elements [c, c + 8) of a row, zeros from `cols` on; any alignment
template <int DT>
__device__ __forceinline__ Raw8<DT> raw_load(const char* row, int c, int cols) {
  constexpr int ES = DT == kInFp32 ? 4 : 2;
  Raw8<DT> r;
  if (c + 8 <= cols) {
    __builtin_memcpy(r.w, __builtin_assume_aligned(row + (size_t)c * ES, ES), sizeof(r.w));
  } else {
#pragma unroll
    for (int i = 0; i < Raw8<DT>::W; ++i) r.w[i] = 0;
    if (ES == 2 && c < cols && cols >= 8) {             // the row's last 16 bytes, moved down: one load
      unsigned __int128 last;
      __builtin_memcpy(&last, row + (size_t)(cols - 8) * ES, 16);
      last >>= (c + 8 - cols) * 16;
      __builtin_memcpy(r.w, &last, 16);
    } else if (c < cols) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c + i < cols) {
          if constexpr (ES == 4) r.w[i] = ((const unsigned int*)row)[c + i];
          else r.w[i >> 1] |= (unsigned int)((const unsigned short*)row)[c + i] << ((i & 1) * 16);
        }
    }
  }
  return r;
}

// |x|'s bits where x is finite, else 0: ordered as the magnitudes are
__device__ __forceinline__ unsigned int finite_bits(float x) {
  const unsigned int b = __builtin_bit_cast(unsigned int, x) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}

constexpr unsigned int kLeastAmax = ((unsigned)(127 - 118) << 23) | 0x600000u;   // 448 * 2^-126 = 1.75 * 2^-118

struct Scale {
  float f;            // float32: the scale; e8m0: 2^e
  int e;              // float32: amax's exponent, -118 to 127; e8m0: e, -126 to 120
  float d;            // float32: amax * 2^-e in [1, 2)
  float m;            // float32: 448 / amax nearly; e8m0: 2^-e (normal numbers either way, so a power of two in them rounds nothing)
};

template <bool E8>
__device__ __forceinline__ Scale make_scale(unsigned int amax) {
  amax = max(amax, kLeastAmax);
  Scale s;
  if constexpr (E8) {
    s.e = (int)(amax >> 23) - 127 - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
    s.f = __builtin_bit_cast(float, (unsigned)(s.e + 127) << 23);
    s.d = 0.f;
    s.m = __builtin_bit_cast(float, (unsigned)(127 - s.e) << 23);
  } else {
    // amax / 448, rounded once: a quotient by 7 with an error under one unit, one correction by its exact remainder
    // (amax / 64 and the results are normal numbers)
    const float a7 = __builtin_bit_cast(float, amax) * 0x1p-6f, q7 = a7 * (1.0f / 7.0f);
    s.f = fmaf(fmaf(-7.0f, q7, a7), 1.0f / 7.0f, q7);
    s.e = (int)(amax >> 23) - 127;
    s.d = __builtin_bit_cast(float, (amax & 0x7fffffu) | 0x3f800000u);
    s.m = ldexpf(448.0f * __builtin_amdgcn_rcpf(s.d), -s.e);
  }
  return s;
}

// Less than kNearBorder where a quotient's last 19 bits are within 8 of zeros, as a border's are.
constexpr unsigned int kNearBorder = 16u << 13;
__device__ __forceinline__ unsigned int border_bits(float y) { return (__builtin_bit_cast(unsigned int, y) + 8) << 13; }

// Any value's quotient: what quantize8 leaves to it.
template <int DT, bool E8>
__device__ __forceinline__ float quotient(float x, const Scale& s) {
  float y = x * s.m;                             // float32 scales: within 4 units in the last place of 448 x / amax
  if constexpr (!E8 && DT != kInFp32) {
    y = __builtin_bit_cast(float, (__builtin_bit_cast(unsigned int, y) + 8) & ~15u);
  } else if constexpr (!E8) {
    if (border_bits(y) < kNearBorder && fabsf(y) >= 0x1p-11f) {   // (under that all are 0) compare with it exactly
      const unsigned int tb = (__builtin_bit_cast(unsigned int, y) + 8) & ~0x7ffffu;
      const double t = (double)__builtin_bit_cast(float, tb) * (double)s.d, n = 448.0 * (double)ldexpf(x, -s.e);
      const double at = fabs(t), an = fabs(n);
      y = __builtin_bit_cast(float, tb + (an > at ? 1u : an < at ? 0xffffffffu : 0u));
    }
  }
  return finite_bits(x) == 0 && x != 0.f ? __builtin_nanf("") : y;
}

// The vector unit is close to the memory's pace here, so a value takes one multiplication, what its type needs at a border,
// and its share of a test for all 8: whether one is not finite (or, of float32, may be a border).
template <int DT, bool E8>
__device__ __forceinline__ qu2 quantize8(const Raw8<DT>& r, bool finite, const Scale& s) {
  float y[8];
  unsigned int near = 0xffffffffu;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    y[i] = raw_get<DT>(r, i) * s.m;
    if constexpr (!E8 && DT == kInFp32) near = min(near, border_bits(y[i]));
    else if constexpr (!E8) y[i] = __builtin_bit_cast(float, (__builtin_bit_cast(unsigned int, y[i]) + 8) & ~15u);
  }
  if (near < kNearBorder || !finite) {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = quotient<DT, E8>(raw_get<DT>(r, i), s);
  }
  qu2 o;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h], y[4 * h + 1], 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h + 2], y[4 * h + 3], w, true);
    o[h] = (unsigned)w;
  }
  return o;
}

__device__ __forceinline__ void store8(unsigned char* row, int c, int cols, qu2 v) {
  if (c + 8 <= cols) {
    __builtin_memcpy(row + c, &v, 8);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < cols) row[c + i] = (unsigned char)(v[i >> 2] >> ((i & 3) * 8));
  }
}

template <bool E8>
__device__ __forceinline__ void store_scale(void* s, size_t at, const Scale& v) {
  if constexpr (E8) ((unsigned char*)s)[at] = (unsigned char)(v.e + 127);
  else ((float*)s)[at] = v.f;
}

// The largest finite magnitude of 8, as a float's bits; whether all are finite. (16-bit magnitudes are ordered as their
// bits are: two to an instruction.)
template <int DT>
__device__ __forceinline__ unsigned int amax8(const Raw8<DT>& r, bool& finite) {
  unsigned int m = 0;
  if constexpr (DT == kInFp32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, r.w[i] & 0x7fffffffu);
    finite = m < 0x7f800000u;
  } else {
    qs2 h = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) h = __builtin_elementwise_max(h, __builtin_bit_cast(qs2, r.w[i] & 0x7fff7fffu));
    const unsigned int top = max(h[0], h[1]);
    finite = top < (DT == kInBf16 ? 0x7f80u : 0x7c00u);
    m = DT == kInBf16 ? top << 16 : __builtin_bit_cast(unsigned int, (float)__builtin_bit_cast(_Float16, (unsigned short)top));
  }
  if (!finite) {
    m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, finite_bits(raw_get<DT>(r, i)));
  }
  return m;
}

// One row's block a quarter wave: 16 lanes of 8 elements; a wave takes 4 U blocks of one row, all loads first.
template <int DT, bool E8, int U>
__global__ void __launch_bounds__(QT) quantize_row_blocks(const QuantArgs a) {
  constexpr int ES = DT == kInFp32 ? 4 : 2;
  const int lane = threadIdx.x & 63, kb_count = (a.cols + 127) / 128, per_row = (kb_count + 4 * U - 1) / (4 * U);
  const unsigned id = blockIdx.x * (QT / 64) + (unsigned)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned row = id / (unsigned)per_row;
  if (row >= (unsigned)a.batches * (unsigned)a.rows) return;
  const int kb0 = (int)(id - row * per_row) * 4 * U + (lane >> 4);
  const unsigned batch = a.batches == 1 ? 0 : row / (unsigned)a.rows, r = row - batch * (unsigned)a.rows;
  const char* x = (const char*)a.x + ((size_t)batch * a.batch_stride + (size_t)r * a.ld) * ES;
  Raw8<DT> v[U];
#pragma unroll
  for (int u = 0; u < U; ++u) v[u] = raw_load<DT>(x, (kb0 + 4 * u) * 128 + (lane & 15) * 8, a.cols);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int kb = kb0 + 4 * u;
    bool finite;
    unsigned int m = amax8<DT>(v[u], finite);
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) m = max(m, (unsigned)__shfl_xor((int)m, d));
    if (kb >= kb_count) continue;
    const Scale s = make_scale<E8>(m);
    store8(a.q + (size_t)row * a.cols, kb * 128 + (lane & 15) * 8, a.cols, quantize8<DT, E8>(v[u], finite, s));
    if ((lane & 15) == 0) store_scale<E8>(a.s, (size_t)row * kb_count + kb, s);
  }
}

// A block of 128 rows a workgroup: thread t holds chunk t & 15 of rows t / 16 + 16 i.
template <int DT, bool E8>
__global__ void __launch_bounds__(QT) quantize_square_blocks(const QuantArgs a) {
  constexpr int ES = DT == kInFp32 ? 4 : 2;
  __shared__ unsigned int part[QT / 64];
  const int kb_count = (a.cols + 127) / 128, rb_count = (a.rows + 127) / 128;
  const int kb = blockIdx.x % kb_count;
  const int rest = blockIdx.x / kb_count, rb = rest % rb_count, batch = rest / rb_count;
  const char* x = (const char*)a.x + (size_t)batch * a.batch_stride * ES;
  const int c = kb * 128 + (threadIdx.x & 15) * 8, r0 = rb * 128 + (threadIdx.x >> 4);
  Raw8<DT> v[8];
  bool finite[8];
  unsigned int m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = r0 + 16 * i;
    v[i] = raw_load<DT>(x + (size_t)(r < a.rows ? r : 0) * a.ld * ES, c, r < a.rows ? a.cols : 0);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, amax8<DT>(v[i], finite[i]));
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) m = max(m, (unsigned)__shfl_xor((int)m, d));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
  __syncthreads();
  m = max(max(part[0], part[1]), max(part[2], part[3]));
  const Scale s = make_scale<E8>(m);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = r0 + 16 * i;
    if (r < a.rows) store8(a.q + ((size_t)batch * a.rows + r) * a.cols, c, a.cols, quantize8<DT, E8>(v[i], finite[i], s));
  }
  if (threadIdx.x == 0) store_scale<E8>(a.s, blockIdx.x, s);
}

template <int DT, bool E8, int U>
int launch_rows(const QuantArgs& a, hipStream_t s) {
  const long long kb = ((long long)a.cols + 127) / 128, waves = (long long)a.batches * a.rows * ((kb + 4 * U - 1) / (4 * U));
  if (waves > 0xffffffffll - QT / 64) return (int)hipErrorInvalidValue;      // (their numbers are 32 bits)
  hipLaunchKernelGGL((quantize_row_blocks<DT, E8, U>), dim3((unsigned)((waves + QT / 64 - 1) / (QT / 64))), dim3(QT), 0, s, a);
  return (int)hipGetLastError();
}

// Two chunks a lane of 16-bit rows that fill the card with waves twice over, one else (16384 x 8192 bf16: 69.9 us, one chunk
// 86.5; 300 rows: 5.1, 4.6; 16384 x 2048 fp32: 32.5, 31.4).
template <int DT, bool E8>
int launch_quant(const QuantArgs& a, hipStream_t s) {
  const long long kb = ((long long)a.cols + 127) / 128;
  if (a.block_rows == 1) {
    if (DT != kInFp32 && (long long)a.batches * a.rows * ((kb + 3) / 4) > 16384) return launch_rows<DT, E8, DT == kInFp32 ? 1 : 2>(a, s);
    return launch_rows<DT, E8, 1>(a, s);
  }
  const long long grid = a.batches * (((long long)a.rows + 127) / 128) * kb;
  if (grid > 0x7fffffff) return (int)hipErrorInvalidValue;
  hipLaunchKernelGGL((quantize_square_blocks<DT, E8>), dim3((unsigned)grid), dim3(QT), 0, s, a);
  return (int)hipGetLastError();
}

// Whether the outputs, which are contiguous, may share memory with x or with each other.
bool may_share(const QuantArgs& a) {
  const __int128 elements = (__int128)a.batches * a.rows * a.cols;
  const __int128 scales = (__int128)a.batches * (((long long)a.rows + a.block_rows - 1) / a.block_rows) * (((long long)a.cols + 127) / 128);
  const MemoryReach x(a.x, elements == 0, (__int128)(a.batches - 1) * a.batch_stride + (__int128)(a.rows - 1) * a.ld + a.cols - 1,
                      a.dtype == kInFp32 ? 4 : 2);
  const MemoryReach q(a.q, elements == 0, elements - 1, 1), s(a.s, elements == 0, scales - 1, a.e8 ? 1 : 4);
  return q.meets(x) || s.meets(x) || q.meets(s);
}

int quantize(const QuantArgs& a, bool look, hipStream_t s) {
  if (a.batches < 0 || a.rows < 0 || a.cols < 0 || (a.block_rows != 1 && a.block_rows != 128)) return (int)hipErrorInvalidValue;
  if (a.rows > 0x7fffffff - 4096 || a.cols > 0x7fffffff - 4096) return (int)hipErrorInvalidValue;      // (indices go past the end)
  if (a.batches == 0 || a.rows == 0 || a.cols == 0) return 0;
  if (look && may_share(a)) return kMayShare;
  switch (a.dtype) {
    case kInBf16: return a.e8 ? launch_quant<kInBf16, true>(a, s) : launch_quant<kInBf16, false>(a, s);
    case kInFp16: return a.e8 ? launch_quant<kInFp16, true>(a, s) : launch_quant<kInFp16, false>(a, s);
    case kInFp32: return a.e8 ? launch_quant<kInFp32, true>(a, s) : launch_quant<kInFp32, false>(a, s);
  }
  return (int)hipErrorInvalidValue;
}

}  // namespace

extern "C" {

int amdgo_quantize_fp8_block(const QuantArgs* args, hipStream_t s) { return args ? quantize(*args, true, s) : (int)hipErrorInvalidValue; }

// The same where the caller knows that the outputs share no memory with x or with each other.
int amdgo_quantize_fp8_block_apart(const QuantArgs* args, hipStream_t s) {
  return args ? quantize(*args, false, s) : (int)hipErrorInvalidValue;
}

}  // extern "C"
