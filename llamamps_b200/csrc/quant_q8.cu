// 8-bit rows: fp16 rows quantised to signed codes with one fp32 scale each,
// alone (the inputs of o_proj and down_proj) or as the output of an RMSNorm
// that may add a residual first.
//
//   s = fp16(residual + x)                     (written out; without a residual s = x)
//   v = s * gamma                              (1 without gamma), exact in fp32: 11 x 11 bits
//   m = max|v|,  r = 1 / sqrt(mean(s^2) + eps) (1 without gamma)
//   code = rint(127 v / m) in [-127, 127],  scale = m r / 127
//
// r cancels in the codes, so the row is read once and held in registers: m and
// the sum of squares come from one reduction.  A zero row has codes and scale
// 0, a row with a NaN or an infinity codes 0 and scale NaN.  127 v / m is one
// rounding of 127 / m and one fused multiply-add that rounds to the integer;
// where that quotient is within 2^-16 of a tie (an element that is half the
// largest is one), the code comes from fp64, so every code is the formula's.
//
// What bounds it: bytes (a row in once, codes and sum out once).
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

constexpr int kCta = 256;                    // threads of a CTA
constexpr float kMagic = 12582912.0f;        // 1.5 * 2^23: adding it rounds to an integer, half to even
constexpr float kNearTie = 0.5f - 1.0f / 65536.0f;

// Over the T threads of a row: the sum of ss and the largest of the bits of m
// (|v| as an unsigned number: a NaN is above infinity).
template <int T>
__device__ __forceinline__ void reduce_row(float& ss, uint32_t& m) {
  ss = warp_sum(ss);
  m = __reduce_max_sync(0xffffffffu, m);
  if constexpr (T > kWarp) {
    __shared__ float rs[T / kWarp];
    __shared__ uint32_t rm[T / kWarp];
    const int warp = threadIdx.x / kWarp;
    if (threadIdx.x % kWarp == 0) {
      rs[warp] = ss;
      rm[warp] = m;
    }
    __syncthreads();
    ss = 0.0f;
    m = 0u;
#pragma unroll
    for (int w = 0; w < T / kWarp; ++w) {
      ss += rs[w];
      m = max(m, rm[w]);
    }
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

// The codes of N elements, as integers in fp32.
template <int N>
__device__ __forceinline__ void row_codes(const float (&v)[N], float inv, uint32_t mbits, float (&c)[N]) {
  float far = 0.0f;  // the largest distance from an integer
#pragma unroll
  for (int i = 0; i < N; ++i) {
    c[i] = fmaf(v[i], inv, kMagic) - kMagic;
    far = fmaxf(far, fabsf(fmaf(v[i], inv, -c[i])));
  }
  if (far > kNearTie) {
    const double m = static_cast<double>(__uint_as_float(mbits));
#pragma unroll
    for (int i = 0; i < N; ++i) c[i] = static_cast<float>(rint(127.0 * static_cast<double>(v[i]) / m));
  }
}

__device__ __forceinline__ uint32_t pack4(const float* c) {
  return (static_cast<uint32_t>(static_cast<int>(c[0])) & 0xFFu) | (static_cast<uint32_t>(static_cast<int>(c[1])) & 0xFFu) << 8 |
         (static_cast<uint32_t>(static_cast<int>(c[2])) & 0xFFu) << 16 | static_cast<uint32_t>(static_cast<int>(c[3])) << 24;
}

__device__ __forceinline__ void unpack8(const uint4& p, float (&f)[8]) {
  const __half2* h = reinterpret_cast<const __half2*>(&p);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __half22float2(h[i]);
    f[2 * i] = t.x, f[2 * i + 1] = t.y;
  }
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  uint4 p;
  __half2* h = reinterpret_cast<__half2*>(&p);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
  return p;
}

// 16-byte pieces of eight elements, T threads a row (32: eight rows a CTA), at most E pieces a thread.
template <int T, int E>
__global__ void __launch_bounds__(kCta) rows_vec_kernel(const RowArgs A) {
  lmps_pdl_trigger();
  lmps_pdl_wait();
  const int t = threadIdx.x % T;
  const size_t row = static_cast<size_t>(blockIdx.x) * (kCta / T) + threadIdx.x / T;
  if (row >= static_cast<size_t>(A.rows)) return;  // (whole warps, or none: T = 256 has a CTA per row)
  const int pieces = A.k / 8;
  const uint4* x = reinterpret_cast<const uint4*>(A.x + row * A.ldx);
  const uint4* gamma = reinterpret_cast<const uint4*>(A.gamma);
  uint4 s[E];
#pragma unroll
  for (int i = 0; i < E; ++i)
    if (t + T * i < pieces) s[i] = x[t + T * i];
  if (A.residual) {
    const uint4* r = reinterpret_cast<const uint4*>(A.residual + row * A.ldr);
    uint4 rv[E];
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (t + T * i < pieces) rv[i] = r[t + T * i];
    uint4* sum = reinterpret_cast<uint4*>(A.sum + row * A.lds);
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (t + T * i < pieces) {
        float a[8], b[8];
        unpack8(s[i], a);
        unpack8(rv[i], b);
#pragma unroll
        for (int e = 0; e < 8; ++e) a[e] += b[e];
        s[i] = pack8(a);
        sum[t + T * i] = s[i];
      }
  }
  float ss = 0.0f;
  uint32_t m = 0u;
#pragma unroll
  for (int i = 0; i < E; ++i)
    if (t + T * i < pieces) {
      float f[8];
      unpack8(s[i], f);
      if (gamma) {
        float g[8];
        unpack8(gamma[t + T * i], g);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          ss = fmaf(f[e], f[e], ss);
          m = max(m, __float_as_uint(f[e] * g[e]) & 0x7FFFFFFFu);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(f[e]) & 0x7FFFFFFFu);
      }
    }
  reduce_row<T>(ss, m);
  float inv, scale;
  row_scale(A, ss, m, inv, scale);
  if (t == 0) A.scales[row] = scale;
  const bool dead = m >= 0x7F800000u;
  uint2* codes = reinterpret_cast<uint2*>(A.codes + row * A.ldc);
  uint4* values = A.values ? reinterpret_cast<uint4*>(A.values + row * A.ldv) : nullptr;
#pragma unroll
  for (int i = 0; i < E; ++i)
    if (t + T * i < pieces) {
      float f[8], c[8];
      unpack8(s[i], f);
      if (gamma) {
        float g[8];
        unpack8(gamma[t + T * i], g);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] *= g[e];
      }
      if (dead)
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = 0.0f;
      row_codes(f, inv, m, c);
      codes[t + T * i] = make_uint2(pack4(c), pack4(c + 4));
      if (values) {
#pragma unroll
        for (int e = 0; e < 8; ++e) c[e] *= scale;
        values[t + T * i] = pack8(c);
      }
    }
}

// Any length, stride and alignment: element t + T i of a row in thread t, the first E of a thread in registers,
// later ones (rows past T E elements) read again, the sum from what this thread wrote.
template <int T, int E>
__global__ void __launch_bounds__(kCta) rows_any_kernel(const RowArgs A) {
  lmps_pdl_trigger();
  lmps_pdl_wait();
  const int t = threadIdx.x % T;
  const size_t row = static_cast<size_t>(blockIdx.x) * (kCta / T) + threadIdx.x / T;
  if (row >= static_cast<size_t>(A.rows)) return;
  const __half* x = A.x + row * A.ldx;
  const __half* r = A.residual ? A.residual + row * A.ldr : nullptr;
  __half* sum = A.residual ? A.sum + row * A.lds : nullptr;
  __half s[E];
#pragma unroll
  for (int i = 0; i < E; ++i) s[i] = t + T * i < A.k ? x[t + T * i] : __half(0.0f);
  if (r) {
    __half b[E];
#pragma unroll
    for (int i = 0; i < E; ++i) b[i] = t + T * i < A.k ? r[t + T * i] : __half(0.0f);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      s[i] = __float2half_rn(__half2float(b[i]) + __half2float(s[i]));
      if (t + T * i < A.k) sum[t + T * i] = s[i];
    }
  }
  float ss = 0.0f;
  uint32_t m = 0u;
  auto take = [&](int i, float f) {
    if (A.gamma) {
      ss = fmaf(f, f, ss);
      f *= __half2float(A.gamma[i]);
    }
    m = max(m, __float_as_uint(f) & 0x7FFFFFFFu);
  };
#pragma unroll
  for (int i = 0; i < E; ++i)
    if (t + T * i < A.k) take(t + T * i, __half2float(s[i]));
  for (int i = t + T * E; i < A.k; i += T) {
    __half v = x[i];
    if (r) {
      v = __float2half_rn(__half2float(r[i]) + __half2float(v));
      sum[i] = v;
    }
    take(i, __half2float(v));
  }
  reduce_row<T>(ss, m);
  float inv, scale;
  row_scale(A, ss, m, inv, scale);
  if (t == 0) A.scales[row] = scale;
  const bool dead = m >= 0x7F800000u;
  int8_t* codes = A.codes + row * A.ldc;
  __half* values = A.values ? A.values + row * A.ldv : nullptr;
  auto give = [&](int i, float f) {
    float v[1] = {A.gamma ? f * __half2float(A.gamma[i]) : f}, c[1];
    if (dead) v[0] = 0.0f;
    row_codes(v, inv, m, c);
    codes[i] = static_cast<int8_t>(static_cast<int>(c[0]));
    if (values) values[i] = __float2half_rn(c[0] * scale);
  };
#pragma unroll
  for (int i = 0; i < E; ++i)
    if (t + T * i < A.k) give(t + T * i, __half2float(s[i]));
  for (int i = t + T * E; i < A.k; i += T) give(i, __half2float(r ? sum[i] : x[i]));
}

template <int T>
static int launch(void (*kernel)(RowArgs), const RowArgs& A, cudaStream_t st) {
  constexpr int per = kCta / T;
  return lmps_launch_pdl(kernel, dim3((A.rows + per - 1) / per), dim3(kCta), 0, st, A);
}

// A warp per row where there are rows enough to fill the GPU and a row fits a warp's registers.
constexpr int kWarpRows = 592;

static int launch_rows(const RowArgs& A, cudaStream_t st) {
  const bool vec = A.k % 8 == 0 && A.ldx % 8 == 0 && A.ldc % 8 == 0 && A.ldr % 8 == 0 && A.lds % 8 == 0 &&
                   A.ldv % 8 == 0 && lmps_aligned(A.x, 16) && lmps_aligned(A.residual, 16) &&
                   lmps_aligned(A.sum, 16) && lmps_aligned(A.gamma, 16) && lmps_aligned(A.codes, 8) &&
                   lmps_aligned(A.values, 16);
  const int pieces = A.k / 8;
  const bool many = A.rows >= kWarpRows;
  if (vec && (many || pieces <= 32) && pieces <= 32 * 8) {
    if (pieces <= 32 * 1) return launch<32>(rows_vec_kernel<32, 1>, A, st);
    if (pieces <= 32 * 3) return launch<32>(rows_vec_kernel<32, 3>, A, st);
    if (pieces <= 32 * 6) return launch<32>(rows_vec_kernel<32, 6>, A, st);
    return launch<32>(rows_vec_kernel<32, 8>, A, st);
  }
  if (vec && pieces <= kCta * 8) {
    if (pieces <= kCta * 1) return launch<kCta>(rows_vec_kernel<kCta, 1>, A, st);
    if (pieces <= kCta * 3) return launch<kCta>(rows_vec_kernel<kCta, 3>, A, st);
    if (pieces <= kCta * 5) return launch<kCta>(rows_vec_kernel<kCta, 5>, A, st);
    return launch<kCta>(rows_vec_kernel<kCta, 8>, A, st);
  }
  if (A.k <= 32 * 16 && (many || A.k <= 64)) return launch<32>(rows_any_kernel<32, 16>, A, st);
  if (A.k <= kCta * 8) return launch<kCta>(rows_any_kernel<kCta, 8>, A, st);
  return launch<kCta>(rows_any_kernel<kCta, 36>, A, st);
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
