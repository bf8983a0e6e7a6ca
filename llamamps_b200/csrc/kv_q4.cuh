// The 4-bit KV cache: its row format, the quantiser of a row, the exact-angle
// RoPE that precedes it, and page lookups with their bounds checks.
//
// One layer's K (and V) pool is uint8 [n_pages, n_kv_heads, page_size * 72].
// A (page, head) block is page_size rows of 64 code bytes (element 2j of the
// 128 in the low nibble of byte j, 2j + 1 in the high one, code + 8: the
// nibble order of the Q4 weights) followed by page_size rows of 4 fp16 scales,
// one per 32 elements.  page_size is a multiple of 16, so codes and scales of
// 16 consecutive positions starting at a multiple of 16 are contiguous runs
// of 1024 and 128 bytes, 16-byte aligned.
//
// Quantiser of a group x[32]: a = max|x|; scale s = the smallest number >= a/7
// with 8 significant bits (a multiple of 2^-24, at most 9344; 1 for a zero
// group); code = rint(x / s), so |code| <= 7.  An 8-bit scale times a 3-bit
// magnitude has at most 11 significant bits: code * s is an fp16 number, so
// readers lose nothing by holding cached values in fp16.  The coarser scale
// costs at most 2^-7 of the quantisation step.  A row with a NaN or infinity
// gets NaN scales: whoever attends to that position gets NaN, nobody else does.
#pragma once

#include "common.cuh"

namespace lmps {
namespace q4 {

constexpr int kDim = 128;       // head dim
constexpr int kGroups = 4;      // scales per row
constexpr int kCodeBytes = 64;  // code bytes per row
constexpr int kRowBytes = 72;   // code bytes + 4 fp16 scales
constexpr int kRun = 16;        // positions per contiguous run (page_size is a multiple)
constexpr int kMaxPage = 1 << 24;  // offsets inside a (page, head) block are 32 bits: 72 * 2^24 < 2^31

// Bits of the int32 error word that the 4-bit cache's kernels raise.
constexpr int kErrTimeout = LMPS_Q4_ERR_TIMEOUT;
constexpr int kErrPage = LMPS_Q4_ERR_PAGE;
constexpr int kErrPosition = LMPS_Q4_ERR_POSITION;

__device__ __forceinline__ void raise_error(int32_t* error, int bits) {
  if (error) atomicOr(error, bits);
}

// The paged pools of one layer as a kernel sees them.
struct Cache {
  const uint8_t* k;
  const uint8_t* v;
  const int32_t* bt;  // [rows, max_pages]
  int n_pages, max_pages, page_size, n_kv;
  int page_shift;  // log2(page_size) when it is a power of two, else -1
  int32_t* error;

  __device__ __forceinline__ int page_index(int p) const { return page_shift >= 0 ? p >> page_shift : p / page_size; }
  // Byte offset of the (page, head) block; `page` in [0, n_pages).
  __device__ __forceinline__ size_t block(int page, int kvh) const {
    return (static_cast<size_t>(page) * n_kv + kvh) * (static_cast<size_t>(page_size) * kRowBytes);
  }
};

static inline int page_shift_of(int page_size) {
  return (page_size & (page_size - 1)) == 0 ? __builtin_ctz(static_cast<unsigned>(page_size)) : -1;
}

// Scale of a group whose largest magnitude is `a` (finite).  a has 11
// significant bits, so a / 7 is either a number of 8 bits or at least 2^-14 of
// itself away from one: the product below, a little above a / 7 by less than
// that, truncates to the largest 8-bit number <= a / 7.
__device__ __forceinline__ float group_scale(float a) {
  if (a == 0.0f) return 1.0f;
  const uint32_t low = __float_as_uint(a * (0.14285714285f * (1.0f + 3.8147e-06f))) & 0xFFFF0000u;  // (2^-18)
  float s = __uint_as_float(__uint_as_float(low) * 7.0f >= a ? low : low + 0x10000u);  // the product is exact
  if (s < 1.52587890625e-05f) s = ceilf(s * 16777216.0f) * 5.9604644775390625e-08f;    // 2^-16: fp16's 2^-24 grid
  return fminf(s, 9344.0f);
}

// 128 / N lanes of a warp quantise one row each: lane l of them holds elements
// N l .. N l + N - 1 (exact fp16 values).  Returns the lane's N nibbles (element
// N l lowest); `scale` is the scale of its group N l / 32.  All lanes take part.
template <int N>
__device__ __forceinline__ uint32_t quantise_row(const float (&x)[N], float& scale) {
  constexpr int kLanes = kDim / N;
  float a = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) a = fmaxf(a, fabsf(x[i]));
  bool finite = a <= 65504.0f;  // (the maximum takes the number where the other is NaN)
#pragma unroll
  for (int i = 0; i < N; ++i) finite = finite && x[i] == x[i];
#pragma unroll
  for (int o = 1; o < kLanes / kGroups; o <<= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
  const uint32_t row = (kLanes == 32 ? 0xffffffffu : (1u << (kLanes & 31)) - 1u) << (threadIdx.x & 31 & ~(kLanes - 1));
  if ((__ballot_sync(0xffffffffu, finite) & row) != row) {
    scale = __int_as_float(0x7FC00000);
    return 0x88888888u >> (32 - 4 * N);
  }
  scale = group_scale(a);
  // x / s by a reciprocal and one residual step (Markstein): exact where the
  // quotient is a number, and it must be where it lies on a tie, which goes to
  // the even code; with 11 bits over 8, other quotients are 2^-12 away from ties.
  // Adding 1.5 * 2^23 rounds to an integer, here code + 8 in the low bits.
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(scale));
  uint32_t w = 0u;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float q = x[i] * r;
    const float c = fmaf(fmaf(-q, scale, x[i]), r, q) + 12582920.0f;
    w |= (__float_as_uint(c) & 0xFu) << (4 * i);
  }
  return w;
}

// cos and sin of pos * inv_freq in fp64, error below 2^-50: the product of a
// position below 2^29 and an fp32 frequency is exact, where an fp32 product is
// off by up to pos * inv_freq * 2^-24 radians (2e-3 at position 32768).  fp64,
// so that K's codes are those of the exactly rotated row: an fp32 rotation
// moves about one code in 10^6 across a rounding border.
// x = k pi/2 + r with pi/2 in two fp64 parts, then the Taylor series of sine and
// cosine on |r| <= pi/4 to r^15 and r^16 (the next terms are below 2^-54).
__device__ __forceinline__ void rope_cos_sin(int pos, float inv_freq, double& c, double& s) {
  const double x = static_cast<double>(pos) * static_cast<double>(inv_freq);
  const double k = rint(x * 0.63661977236758134308);
  double r = fma(-k, 1.57079632679489655800, x);
  r = fma(-k, 6.12323399573676603587e-17, r);
  const double z = r * r;
  double ps = -1.0 / 1307674368000.0, pc = 1.0 / 20922789888000.0;
  ps = fma(ps, z, 1.0 / 6227020800.0);
  pc = fma(pc, z, -1.0 / 87178291200.0);
  ps = fma(ps, z, -1.0 / 39916800.0);
  pc = fma(pc, z, 1.0 / 479001600.0);
  ps = fma(ps, z, 1.0 / 362880.0);
  pc = fma(pc, z, -1.0 / 3628800.0);
  ps = fma(ps, z, -1.0 / 5040.0);
  pc = fma(pc, z, 1.0 / 40320.0);
  ps = fma(ps, z, 1.0 / 120.0);
  pc = fma(pc, z, -1.0 / 720.0);
  ps = fma(ps, z, -1.0 / 6.0);
  pc = fma(pc, z, 1.0 / 24.0);
  pc = fma(pc, z, -0.5);
  const double sn = fma(r * z, ps, r), cn = fma(pc, z, 1.0);
  const int q = static_cast<int>(static_cast<long long>(k)) & 3;
  const double a = (q & 1) ? sn : cn, b = (q & 1) ? cn : sn;  // cos, sin up to their signs
  c = (q == 1 || q == 2) ? -a : a;
  s = (q >= 2) ? -b : b;
}

// (x1, x2) -> (x1 c - x2 s, x1 s + x2 c), fp64 rounded through fp32 to fp16.
__device__ __forceinline__ void rope_rotate64(__half& a, __half& b, double c, double s) {
  const double x1 = static_cast<double>(__half2float(a)), x2 = static_cast<double>(__half2float(b));
  a = __float2half_rn(static_cast<float>(__fma_rn(x1, c, -__dmul_rn(x2, s))));
  b = __float2half_rn(static_cast<float>(__fma_rn(x1, s, __dmul_rn(x2, c))));
}
// The same in fp32, from cos and sin rounded to fp32: q, which no rounding
// border waits for, is off by at most 3 * 2^-24 (|x1| + |x2|) before it is
// rounded to fp16.  (Explicit operations: every kernel gets the same bits.)
__device__ __forceinline__ void rope_rotate32(float x1, float x2, float2 cs, float& y1, float& y2) {
  y1 = __fmaf_rn(x1, cs.x, -__fmul_rn(x2, cs.y));
  y2 = __fmaf_rn(x1, cs.y, __fmul_rn(x2, cs.x));
}

__device__ __forceinline__ void rope_rotate_by(__half& a, __half& b, const double2& t) { rope_rotate64(a, b, t.x, t.y); }
__device__ __forceinline__ void rope_rotate_by(__half& a, __half& b, const float2& t) {
  float y1, y2;
  rope_rotate32(__half2float(a), __half2float(b), t, y1, y2);
  a = __float2half_rn(y1);
  b = __float2half_rn(y2);
}
// One of the two: the first (x = x1, other = x2) or the second (x = x2, other = x1), the same operations.
__device__ __forceinline__ __half rope_rotate_one(__half x, __half other, bool first, const double2& t) {
  const double o = static_cast<double>(__half2float(x)), p = static_cast<double>(__half2float(other));
  const double m = __dmul_rn(first ? p : o, first ? t.y : t.x);
  return __float2half_rn(static_cast<float>(__fma_rn(first ? o : p, first ? t.x : t.y, first ? -m : m)));
}
__device__ __forceinline__ __half rope_rotate_one(__half x, __half other, bool first, const float2& t) {
  const float o = __half2float(x), p = __half2float(other);
  const float m = __fmul_rn(first ? p : o, first ? t.y : t.x);
  return __float2half_rn(__fmaf_rn(first ? o : p, first ? t.x : t.y, first ? -m : m));
}
// 128 / N lanes of a warp rotate one head's row each in place: lane l of them holds elements N l .. N l + N - 1;
// cs: 64 (cos, sin), fp64 for K and fp32 for q.
template <int N, class Pair>
__device__ __forceinline__ void rotate_head(__half (&x)[N], const Pair* cs, int style, int lane) {
  constexpr int kHalf = kDim / 2 / N;  // lanes of half a row
  if (style == LMPS_ROPE_INTERLEAVED) {
    const int l = lane & (2 * kHalf - 1);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) rope_rotate_by(x[2 * i], x[2 * i + 1], cs[N / 2 * l + i]);
  } else {  // element j pairs with j + 64: the partner lane is half a row away
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const unsigned other = __shfl_xor_sync(0xffffffffu, static_cast<unsigned>(__half_as_ushort(x[i])), kHalf);
      x[i] = rope_rotate_one(x[i], __ushort_as_half(static_cast<unsigned short>(other)), (lane & kHalf) == 0,
                             cs[N * (lane & (kHalf - 1)) + i]);
    }
  }
}

}  // namespace q4
}  // namespace lmps
