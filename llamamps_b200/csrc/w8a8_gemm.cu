// W8A8: 8-bit rows (a token's codes and its scale) times 8-bit weights (a
// channel's codes and its scale), exact 32-bit integer sums:
//
//   y[t][c] = fp16(x_scale[t] w_scale[c] sum_k x[t][k] w[c][k] + bias[c] + residual[t][c])
//   gated:   y[t][c] = fp16(silu(g) u) with g from weight row c, u from row n + c
//
// The sum of up to 131071 products of codes fits 32 bits; everything after it
// is fp32 and rounded once.
#include "common.cuh"

namespace lmps {
namespace w8 {

constexpr int kMaxK = 131071;  // 2^31 / 2^14: codes of -128 included

struct Args {
  const int8_t* x;
  size_t ldx;
  const float* xs;
  const int8_t* w;
  size_t ldw;
  const float* ws;
  const __half* bias;
  const __half* residual;
  size_t ldr;
  __half* y;
  size_t ldy;
  int m, n, k, swiglu;
};

// y[t][c] from the integer sum(s) and the scales.
__device__ __forceinline__ float linear_value(int acc, float xs, float ws) { return static_cast<float>(acc) * xs * ws; }

// A warp per output channel and four tokens, lanes over K, four products a
// dp4a: for single tokens, where the weights' bytes are all there is.
constexpr int kTokens = 4;
constexpr int kGemvWarps = 4;

template <bool GATED>
__global__ void __launch_bounds__(kGemvWarps* kWarp) gemv_kernel(const Args A) {
  lmps_pdl_trigger();
  lmps_pdl_wait();
  const int c = blockIdx.x * kGemvWarps + static_cast<int>(threadIdx.x / kWarp), lane = threadIdx.x % kWarp;
  const int t0 = blockIdx.y * kTokens;
  if (c >= A.n) return;
  const int8_t* w0 = A.w + static_cast<size_t>(c) * A.ldw;
  const int8_t* w1 = w0 + static_cast<size_t>(A.n) * A.ldw;
  const int whole = A.k / 16;
  int acc[2][kTokens] = {};
  for (int j = lane; j < whole; j += kWarp) {
    const int4 a = *reinterpret_cast<const int4*>(w0 + 16 * j);
    const int4 b = GATED ? *reinterpret_cast<const int4*>(w1 + 16 * j) : make_int4(0, 0, 0, 0);
#pragma unroll
    for (int t = 0; t < kTokens; ++t) {
      if (t0 + t >= A.m) break;
      const int4 v = *reinterpret_cast<const int4*>(A.x + static_cast<size_t>(t0 + t) * A.ldx + 16 * j);
      acc[0][t] = __dp4a(a.x, v.x, __dp4a(a.y, v.y, __dp4a(a.z, v.z, __dp4a(a.w, v.w, acc[0][t]))));
      if (GATED) acc[1][t] = __dp4a(b.x, v.x, __dp4a(b.y, v.y, __dp4a(b.z, v.z, __dp4a(b.w, v.w, acc[1][t]))));
    }
  }
  if (16 * whole + lane < A.k) {  // the last k % 16 elements
    const int i = 16 * whole + lane;
#pragma unroll
    for (int t = 0; t < kTokens; ++t) {
      if (t0 + t >= A.m) break;
      const int v = A.x[static_cast<size_t>(t0 + t) * A.ldx + i];
      acc[0][t] += w0[i] * v;
      if (GATED) acc[1][t] += w1[i] * v;
    }
  }
#pragma unroll
  for (int t = 0; t < kTokens; ++t) {
    if (t0 + t >= A.m) break;
    const int a = __reduce_add_sync(0xffffffffu, acc[0][t]);
    const int b = GATED ? __reduce_add_sync(0xffffffffu, acc[1][t]) : 0;
    if (lane != 0) continue;
    const size_t row = static_cast<size_t>(t0 + t);
    float v = linear_value(a, A.xs[row], A.ws[c]);
    if (GATED) v = silu_mul(v, linear_value(b, A.xs[row], A.ws[A.n + c]));
    if (A.bias) v += __half2float(A.bias[c]);
    if (A.residual) v += __half2float(A.residual[row * A.ldr + c]);
    A.y[row * A.ldy + c] = __float2half_rn(v);
  }
}

}  // namespace w8
}  // namespace lmps

using namespace lmps;

extern "C" int lmps_w8a8_gemm(const int8_t* x, int ldx, const float* x_scales, const int8_t* w, int ldw,
                              const float* w_scales, const uint16_t* bias, const uint16_t* residual, int ldr,
                              uint16_t* y, int ldy, int m, int n, int k, int swiglu, int32_t* error, void* stream) {
  LMPS_CHECK_ARG(x && x_scales && w && w_scales && y && error);
  LMPS_CHECK_ARG(m >= 1 && n >= 1 && k >= 1 && (swiglu == 0 || swiglu == 1));
  LMPS_CHECK_ARG(ldx >= k && ldx % 16 == 0 && ldw >= k && ldw % 16 == 0 && ldy >= n);
  LMPS_CHECK_ARG(!residual || ldr >= n);
  LMPS_CHECK_ARG(!swiglu || (!bias && !residual));
  LMPS_CHECK_ARG(lmps_aligned(x, 16) && lmps_aligned(w, 16) && lmps_aligned(x_scales, 4) && lmps_aligned(w_scales, 4));
  LMPS_CHECK_ARG(lmps_aligned(y, 2) && lmps_aligned(bias, 2) && lmps_aligned(residual, 2) && lmps_aligned(error, 4));
  if (k > w8::kMaxK || n > (1 << 30)) return LMPS_ERR_UNSUPPORTED;
  w8::Args A{};
  A.x = x;
  A.ldx = static_cast<size_t>(ldx);
  A.xs = x_scales;
  A.w = w;
  A.ldw = static_cast<size_t>(ldw);
  A.ws = w_scales;
  A.bias = reinterpret_cast<const __half*>(bias);
  A.residual = reinterpret_cast<const __half*>(residual);
  A.ldr = static_cast<size_t>(residual ? ldr : 0);
  A.y = reinterpret_cast<__half*>(y);
  A.ldy = static_cast<size_t>(ldy);
  A.m = m;
  A.n = n;
  A.k = k;
  A.swiglu = swiglu;
  const dim3 grid((n + w8::kGemvWarps - 1) / w8::kGemvWarps, (m + w8::kTokens - 1) / w8::kTokens);
  if (grid.y > 65535u) return LMPS_ERR_UNSUPPORTED;
  return lmps_launch_pdl(swiglu ? w8::gemv_kernel<true> : w8::gemv_kernel<false>, grid,
                         dim3(w8::kGemvWarps * kWarp), 0, lmps_stream(stream), A);
}
