// 8-bit rows: fp16 rows quantised to signed codes with one fp32 scale each,
// alone (the inputs of o_proj and down_proj) or as the output of an RMSNorm
// that may add a residual first.
//
//   s = fp16(residual + x)                     (written out; without a residual s = x)
//   v = s * gamma                              (1 without gamma), exact in fp32: 11 x 11 bits
//   m = max|v|,  r = 1 / sqrt(mean(s^2) + eps) (1 without gamma)
//   code = rint(127 v / m) in [-127, 127],  scale = m r / 127
//
// r cancels in the codes, so the row is read once: m and the sum of squares
// come from one block reduction.  A zero row has codes and scale 0, a row with
// a NaN or an infinity codes 0 and scale NaN.  127 v / m is one rounding of
// 127 / m and one fused multiply-add that rounds to the integer, so a code is
// the formula's unless the quotient is within 2^-16 of a tie.
#include "common.cuh"

namespace lmps {
namespace q8 {

struct RowArgs {
  const __half* x;
  size_t ldx;
  const __half* residual;
  size_t ldr;
  __half* sum;
  size_t lds;
  const __half* gamma;
  int8_t* codes;
  size_t ldc;
  float* scales;
  __half* values;
  size_t ldv;
  int rows, k;
  float eps;
};

constexpr int kThreads = 256;

// Of all threads of the row: the sum of ss and the largest of the bits of m
// (|v| as an unsigned number: a NaN is above infinity).
__device__ __forceinline__ void block_reduce(float& ss, uint32_t& m) {
  __shared__ float rs[kThreads / kWarp];
  __shared__ uint32_t rm[kThreads / kWarp];
  const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;
  ss = warp_sum(ss);
  m = __reduce_max_sync(0xffffffffu, m);
  if (lane == 0) {
    rs[warp] = ss;
    rm[warp] = m;
  }
  __syncthreads();
  ss = 0.0f;
  m = 0u;
#pragma unroll
  for (int w = 0; w < kThreads / kWarp; ++w) {
    ss += rs[w];
    m = max(m, rm[w]);
  }
}

// The factor of the codes and the scale of a row.
__device__ __forceinline__ void row_scale(const RowArgs& A, float ss, uint32_t mbits, float& inv, float& scale) {
  const float m = __uint_as_float(mbits);
  const float r = A.gamma ? 1.0f / sqrtf(ss / static_cast<float>(A.k) + A.eps) : 1.0f;
  inv = 127.0f / m;
  scale = m * r / 127.0f;
  if (mbits == 0u) inv = scale = 0.0f;
  if (mbits >= 0x7F800000u) {
    inv = 0.0f;
    scale = __uint_as_float(0x7FC00000u);
  }
}

// rint(v * inv) for |v * inv| < 2^21: the low byte of the sum with 1.5 * 2^23.
__device__ __forceinline__ uint32_t code_bits(float v, float inv) {
  return __float_as_uint(fmaf(v, inv, 12582912.0f));
}
__device__ __forceinline__ float code_value(uint32_t bits) { return __uint_as_float(bits) - 12582912.0f; }

// Any length, stride and alignment: a CTA per row, one element a time.
__global__ void __launch_bounds__(kThreads) rows_kernel(const RowArgs A) {
  lmps_pdl_trigger();
  lmps_pdl_wait();
  const size_t row = blockIdx.x;
  const __half* x = A.x + row * A.ldx;
  const __half* s = x;
  if (A.residual) {
    s = A.sum + row * A.lds;
    for (int i = threadIdx.x; i < A.k; i += kThreads)
      A.sum[row * A.lds + i] = __float2half_rn(__half2float(A.residual[row * A.ldr + i]) + __half2float(x[i]));
  }
  float ss = 0.0f;
  uint32_t m = 0u;
  for (int i = threadIdx.x; i < A.k; i += kThreads) {
    const float f = __half2float(s[i]);
    const float v = A.gamma ? f * __half2float(A.gamma[i]) : f;
    ss = fmaf(f, f, ss);
    m = max(m, __float_as_uint(v) & 0x7FFFFFFFu);
  }
  block_reduce(ss, m);
  float inv, scale;
  row_scale(A, ss, m, inv, scale);
  if (threadIdx.x == 0) A.scales[row] = scale;
  const bool dead = m >= 0x7F800000u;
  for (int i = threadIdx.x; i < A.k; i += kThreads) {
    float v = __half2float(s[i]);
    if (A.gamma) v *= __half2float(A.gamma[i]);
    const uint32_t c = code_bits(dead ? 0.0f : v, inv);
    A.codes[row * A.ldc + i] = static_cast<int8_t>(c & 0xFFu);
    if (A.values) A.values[row * A.ldv + i] = __float2half_rn(code_value(c) * scale);
  }
}

static int launch_rows(const RowArgs& A, cudaStream_t st) {
  return lmps_launch_pdl(rows_kernel, dim3(A.rows), dim3(kThreads), 0, st, A);
}

}  // namespace q8
}  // namespace lmps

using namespace lmps;

static const __half* CH(const uint16_t* p) { return reinterpret_cast<const __half*>(p); }
static __half* H(uint16_t* p) { return reinterpret_cast<__half*>(p); }

extern "C" int lmps_quantise_rows_q8(const uint16_t* x, int ldx, int8_t* codes, int ldc, float* scales,
                                     uint16_t* values, int ldv, int rows, int k, void* stream) {
  LMPS_CHECK_ARG(x && codes && scales);
  LMPS_CHECK_ARG(rows >= 1 && k >= 1 && ldx >= k && ldc >= k && (!values || ldv >= k));
  LMPS_CHECK_ARG(lmps_aligned(x, 2) && lmps_aligned(scales, 4) && lmps_aligned(values, 2));
  q8::RowArgs A{};
  A.x = CH(x);
  A.ldx = static_cast<size_t>(ldx);
  A.codes = codes;
  A.ldc = static_cast<size_t>(ldc);
  A.scales = scales;
  A.values = H(values);
  A.ldv = static_cast<size_t>(values ? ldv : 0);
  A.rows = rows;
  A.k = k;
  return q8::launch_rows(A, lmps_stream(stream));
}

extern "C" int lmps_rms_norm_q8(const uint16_t* x, int ldx, const uint16_t* residual, int ldr, uint16_t* sum, int lds,
                                const uint16_t* gamma, float eps, int8_t* codes, int ldc, float* scales,
                                uint16_t* values, int ldv, int rows, int k, void* stream) {
  LMPS_CHECK_ARG(x && gamma && codes && scales && eps >= 0.0f);
  LMPS_CHECK_ARG(rows >= 1 && k >= 1 && ldx >= k && ldc >= k && (!values || ldv >= k));
  LMPS_CHECK_ARG(!residual == !sum && (!residual || (ldr >= k && lds >= k)));
  LMPS_CHECK_ARG(lmps_aligned(x, 2) && lmps_aligned(residual, 2) && lmps_aligned(sum, 2) && lmps_aligned(gamma, 2) &&
                 lmps_aligned(scales, 4) && lmps_aligned(values, 2));
  q8::RowArgs A{};
  A.x = CH(x);
  A.ldx = static_cast<size_t>(ldx);
  A.residual = CH(residual);
  A.ldr = static_cast<size_t>(residual ? ldr : 0);
  A.sum = H(sum);
  A.lds = static_cast<size_t>(sum ? lds : 0);
  A.gamma = CH(gamma);
  A.eps = eps;
  A.codes = codes;
  A.ldc = static_cast<size_t>(ldc);
  A.scales = scales;
  A.values = H(values);
  A.ldv = static_cast<size_t>(values ? ldv : 0);
  A.rows = rows;
  A.k = k;
  return q8::launch_rows(A, lmps_stream(stream));
}
