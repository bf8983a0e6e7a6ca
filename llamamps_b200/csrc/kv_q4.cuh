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

// Scale of a group whose largest magnitude is `a` (finite).  a / 7 is rounded
// up to 24 bits and that up to 8 (the low 16 of fp32's 24): rounding up twice
// on nested grids is rounding up once.
__device__ __forceinline__ float group_scale(float a) {
  if (a == 0.0f) return 1.0f;
  float s = __uint_as_float((__float_as_uint(__fdiv_ru(a, 7.0f)) + 0xFFFFu) & 0xFFFF0000u);
  if (s < 1.52587890625e-05f) s = ceilf(s * 16777216.0f) * 5.9604644775390625e-08f;  // 2^-16: fp16's 2^-24 grid
  return fminf(s, 9344.0f);
}

// A warp quantises one row: lane l holds elements 4l .. 4l+3 (exact fp16
// values).  Returns the lane's four nibbles (element 4l lowest: bytes 2l and
// 2l + 1 of the row); `scale` is the scale of its group l / 8.
__device__ __forceinline__ uint32_t quantise_row(const float (&x)[4], float& scale) {
  float a = 0.0f;
  bool finite = true;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    a = fmaxf(a, fabsf(x[i]));
    finite = finite && fabsf(x[i]) <= 65504.0f;
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
  if (!__all_sync(0xffffffffu, finite)) {
    scale = __int_as_float(0x7FC00000);
    return 0x8888u;
  }
  scale = group_scale(a);
  uint32_t w = 0u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // IEEE division: x / s may lie on a tie, which rint sends to the even code
    const float c = fminf(fmaxf(rintf(__fdiv_rn(x[i], scale)), -7.0f), 7.0f);
    w |= static_cast<uint32_t>(static_cast<int>(c) + 8) << (4 * i);
  }
  return w;
}

// cos and sin of pos * inv_freq: the product of a position below 2^29 and an
// fp32 frequency is exact in fp64, where an fp32 product is off by up to
// pos * inv_freq * 2^-24 radians (2e-3 at position 32768).  fp64 throughout,
// so that K's codes are those of the exactly rotated row: an fp32 rotation
// moves about one code in 10^6 across a rounding border.
__device__ __forceinline__ void rope_cos_sin(int pos, float inv_freq, double& c, double& s) {
  sincos(static_cast<double>(pos) * static_cast<double>(inv_freq), &s, &c);
}

// (x1, x2) -> (x1 c - x2 s, x1 s + x2 c), fp64 rounded through fp32 to fp16.
__device__ __forceinline__ void rope_rotate64(__half& a, __half& b, double c, double s) {
  const double x1 = static_cast<double>(__half2float(a)), x2 = static_cast<double>(__half2float(b));
  a = __float2half_rn(static_cast<float>(x1 * c - x2 * s));
  b = __float2half_rn(static_cast<float>(x1 * s + x2 * c));
}

// A warp rotates one head's row in place: lane l holds elements 4l .. 4l+3.
__device__ __forceinline__ void rotate_head(__half (&x)[4], const double2* cs, int style, int lane) {
  if (style == LMPS_ROPE_INTERLEAVED) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const double2 t = cs[2 * lane + i];
      rope_rotate64(x[2 * i], x[2 * i + 1], t.x, t.y);
    }
  } else {  // element j pairs with j + 64: the partner lane is 16 away
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const double2 t = cs[4 * (lane & 15) + i];
      const unsigned other = __shfl_xor_sync(0xffffffffu, static_cast<unsigned>(__half_as_ushort(x[i])), 16);
      const __half p = __ushort_as_half(static_cast<unsigned short>(other));
      __half a = lane < 16 ? x[i] : p, b = lane < 16 ? p : x[i];
      rope_rotate64(a, b, t.x, t.y);
      x[i] = lane < 16 ? a : b;
    }
  }
}

}  // namespace q4
}  // namespace lmps
