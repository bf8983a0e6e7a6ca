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
// division of two ulp and one fused multiply-add that rounds to the integer;
// where that quotient is within rounding of a tie h (an element that is half
// the largest is one), the sign of 127 v - h m decides, which two products and
// what they lost give exactly, so every code is the formula's, whatever the
// call.  The norm's scales differ in their last bits between calls of different
// size: the squares are added in the order of the threads that a row has.
//
// Bound by bytes (a row in once, codes and sum out once) where there are many:
// 16384 x 8960 64 us (6.9 TB/s; with the values 107, 6.8 TB/s), norm of 16384 x
// 1536 with residual 29 us (6.1 TB/s); by instructions without one, 18.3 us (4.1
// TB/s: a thread's six products with gamma are made twice).  A row's latency else:
// 64 x 8960 1.9 us, norm of 64 x 1536 with residual 2.0 (in a graph of 200 calls).
#include <type_traits>

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

constexpr int kMaxK = 1 << 30;  // positions in a row, and the steps past its end, fit 32 bits
constexpr int kCta = 256;  // threads of a CTA, but where a row has more
template <int T>
constexpr int kCtaOf = T > kCta ? T : kCta;
constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23: adding it rounds to an integer, half to even, in the low bits
constexpr float kNearTie = 0.5f - 3.2e-5f;  // (127 / m is off by 2^-22 of itself, so a quotient by 127 x 2^-22 = 3.1e-5)

// The largest of m, |a| and |b| (a NaN stays).
__device__ __forceinline__ float max_abs(float m, float a, float b) {
  asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(a), "f"(b));
  return m;
}
// Two fp32 operations at once.
__device__ __forceinline__ uint64_t pair2(float a, float b) {
  uint64_t p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
  return p;
}
__device__ __forceinline__ float2 both(uint64_t p) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p));
  return f;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}

// Over the T threads of a row: the largest m (|v|; a NaN stays) as its bits, and with SUM the sum of ss, which only
// the threads get that `want` it (whole warps).
template <int T, bool SUM>
__device__ __forceinline__ void reduce_row(float& ss, float m, uint32_t& mbits, bool want) {
  if constexpr (SUM) ss = warp_sum(ss);
  mbits = __reduce_max_sync(0xffffffffu, __float_as_uint(m) & 0x7FFFFFFFu);  // (a NaN's bits are above infinity's)
  if constexpr (T > kWarp) {
    constexpr int kWarps = T / kWarp;
    __shared__ float rs[kCtaOf<T> / kWarp];
    __shared__ uint32_t rm[kCtaOf<T> / kWarp];
    const int warp = threadIdx.x / kWarp, first = warp / kWarps * kWarps;
    if (threadIdx.x % kWarp == 0) {
      if constexpr (SUM) rs[warp] = ss;
      rm[warp] = mbits;
    }
    asm volatile("bar.sync %0, %1;" ::"r"(1 + first / kWarps), "n"(T) : "memory");
    if constexpr (kWarps <= 4) {
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mbits = max(mbits, rm[first + w]);
    } else {
      mbits = __reduce_max_sync(0xffffffffu, rm[first + threadIdx.x % kWarps]);
    }
    if (SUM && want) {
      ss = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) ss += rs[first + w];
    }
  }
}

// The factor of the codes, and the scale of a row.
__device__ __forceinline__ float row_factor(uint32_t mbits) {
  return mbits == 0u || mbits >= 0x7F800000u ? 0.0f : __fdividef(127.0f, __uint_as_float(mbits));
}
__device__ __forceinline__ float row_scale(const RowArgs& A, float ss, uint32_t mbits) {
  const float r = A.gamma ? 1.0f / sqrtf(ss / static_cast<float>(A.k) + A.eps) : 1.0f;
  if (mbits >= 0x7F800000u) return __uint_as_float(0x7FC00000u);
  return mbits == 0u ? 0.0f : __uint_as_float(mbits) * r / 127.0f;
}

// The codes of eight elements, in the low bytes of t (and as t - kMagic).
__device__ __forceinline__ void row_codes(const float (&v)[8], float inv, uint32_t mbits, float (&t)[8]) {
  const uint64_t inv2 = pair2(inv, inv), magic2 = pair2(kMagic, kMagic), minus2 = pair2(-1.0f, -1.0f);
  float far = 0.0f;  // the largest distance of a quotient from its code
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const uint64_t v2 = pair2(v[i], v[i + 1]), t2 = fma2(v2, inv2, magic2);
    const float2 f = both(t2), d = both(fma2(v2, inv2, fma2(t2, minus2, magic2)));
    t[i] = f.x, t[i + 1] = f.y;
    far = max_abs(far, d.x, d.y);
  }
  if (far > kNearTie) {
    const float m = __uint_as_float(mbits);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float c = t[i] - kMagic, h = c + copysignf(0.5f, fmaf(v[i], inv, -c));
      // With |127 v| < 2^e and v, m of 22 bits all four are multiples of 2^(e - 31).  Next to the tie p - q is exact, and
      // lp - lq, at most 2^(e - 23), as well; away from it the sign is p - q's.
      const float p = __fmul_rn(127.0f, v[i]), q = __fmul_rn(h, m), lp = fmaf(127.0f, v[i], -p), lq = fmaf(h, m, -q);
      const float above = (p - q) + (lp - lq);
      t[i] = (above == 0.0f ? h : above > 0.0f ? h + 0.5f : h - 0.5f) + kMagic;
    }
  }
}

__device__ __forceinline__ uint32_t pack4(const float* t) {  // four low bytes
  return __byte_perm(__byte_perm(__float_as_uint(t[0]), __float_as_uint(t[1]), 0x0040),
                     __byte_perm(__float_as_uint(t[2]), __float_as_uint(t[3]), 0x0040), 0x5410);
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

// 16-byte pieces of eight elements, T threads a row, at most E pieces a thread.  GAMMA: the norm's rows.  Up to three
// pieces a thread keeps their products with gamma, else it makes them again.
template <int T, int E, bool GAMMA>
__global__ void __launch_bounds__(kCtaOf<T>) rows_vec_kernel(const RowArgs A) {
  lmps_pdl_trigger();
  lmps_pdl_wait();
  const int t = threadIdx.x % T;
  const size_t row = static_cast<size_t>(blockIdx.x) * (kCtaOf<T> / T) + threadIdx.x / T;
  if (row >= static_cast<size_t>(A.rows)) return;  // (all T threads of the row)
  const int pieces = A.k / 8;
  const uint4* x = reinterpret_cast<const uint4*>(A.x + row * A.ldx);
  const uint4* gamma = reinterpret_cast<const uint4*>(A.gamma);
  uint4 s[E];
#pragma unroll
  for (int i = 0; i < E; ++i)
    if (t + T * i < pieces) s[i] = x[t + T * i];
  if (GAMMA && A.residual) {
    const uint4* r = reinterpret_cast<const uint4*>(A.residual + row * A.ldr);
    uint4 rv[E];
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (t + T * i < pieces) rv[i] = r[t + T * i];
    uint4* sum = reinterpret_cast<uint4*>(A.sum + row * A.lds);
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (t + T * i < pieces) {
        __half2* a = reinterpret_cast<__half2*>(&s[i]);
        const __half2* b = reinterpret_cast<const __half2*>(&rv[i]);
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = __hadd2_rn(a[e], b[e]);
        sum[t + T * i] = s[i];
      }
  }
  constexpr bool kHold = GAMMA && E <= 3;
  uint64_t held[kHold ? E : 1][4];  // two elements each
  // the products of piece i with gamma
  auto products = [&](int i, uint64_t (&v)[4], auto&& each) {
    const __half2 *h = reinterpret_cast<const __half2*>(&s[i]);
    const uint4 gp = gamma[t + T * i];
    const __half2* g = reinterpret_cast<const __half2*>(&gp);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = __half22float2(h[e]), w = __half22float2(g[e]);
      const uint64_t f2 = pair2(f.x, f.y);
      v[e] = mul2(f2, pair2(w.x, w.y));
      each(f2, v[e]);
    }
  };
  float ss = 0.0f, m = 0.0f;
  if constexpr (GAMMA) {
    uint64_t ss2 = 0;
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (t + T * i < pieces)
        products(i, held[kHold ? i : 0], [&](uint64_t f2, uint64_t v2) {
          ss2 = fma2(f2, f2, ss2);
          const float2 v = both(v2);
          m = max_abs(m, v.x, v.y);
        });
    const float2 f = both(ss2);
    ss = f.x + f.y;
  } else {
    __half2 m2 = __float2half2_rn(0.0f);
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (t + T * i < pieces) {
        const __half2* h = reinterpret_cast<const __half2*>(&s[i]);
#pragma unroll
        for (int e = 0; e < 4; ++e) m2 = __hmax2_nan(m2, __habs2(h[e]));
      }
    m = max_abs(0.0f, __low2float(m2), __high2float(m2));
  }
  const bool scaling = A.values || t < kWarp;
  uint32_t mbits;
  reduce_row<T, GAMMA>(ss, m, mbits, scaling);
  float scale = 0.0f;
  if (scaling) scale = row_scale(A, ss, mbits);
  if (t == 0) A.scales[row] = scale;
  uint2* codes = reinterpret_cast<uint2*>(A.codes + row * A.ldc);
  uint4* values = A.values ? reinterpret_cast<uint4*>(A.values + row * A.ldv) : nullptr;
  if (mbits >= 0x7F800000u) {  // (codes 0, values NaN)
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (t + T * i < pieces) {
        codes[t + T * i] = make_uint2(0u, 0u);
        if (values) values[t + T * i] = make_uint4(0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu);
      }
    return;
  }
  const float inv = row_factor(mbits);
#pragma unroll
  for (int i = 0; i < E; ++i)
    if (t + T * i < pieces) {
      float f[8], c[8];
      if constexpr (GAMMA) {
        if constexpr (!kHold) products(i, held[0], [](uint64_t, uint64_t) {});
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 v = both(held[kHold ? i : 0][e]);
          f[2 * e] = v.x, f[2 * e + 1] = v.y;
        }
      } else {
        unpack8(s[i], f);
      }
      row_codes(f, inv, mbits, c);
      codes[t + T * i] = make_uint2(pack4(c), pack4(c + 4));
      if (values) {
#pragma unroll
        for (int e = 0; e < 8; ++e) c[e] = (c[e] - kMagic) * scale;
        values[t + T * i] = pack8(c);
      }
    }
}

// Any length, stride and alignment: element t + T i of a row in thread t, the first 8 E of a thread in registers,
// later ones (rows past 8 T E elements) read again, the sum from what this thread wrote.
template <int T, int E>
__global__ void __launch_bounds__(kCtaOf<T>) rows_any_kernel(const RowArgs A) {
  lmps_pdl_trigger();
  lmps_pdl_wait();
  const int t = threadIdx.x % T;
  const size_t row = static_cast<size_t>(blockIdx.x) * (kCtaOf<T> / T) + threadIdx.x / T;
  if (row >= static_cast<size_t>(A.rows)) return;
  const __half* x = A.x + row * A.ldx;
  const __half* r = A.residual ? A.residual + row * A.ldr : nullptr;
  __half* sum = A.residual ? A.sum + row * A.lds : nullptr;
  const __half none = __ushort_as_half(0);
  // (eight elements that are all in the row go without the checks)
  auto each = [&](int base, auto&& f) {
    if (base + 7 * T < A.k) f(std::true_type{});
    else if (base < A.k) f(std::false_type{});
  };
  // elements base + T j for j < 8 (zero past the row); the sum is written on the way
  auto load8 = [&](auto whole, int base, __half (&s)[8]) {
    auto in = [&](int j) { return whole() || base + T * j < A.k; };
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] = in(j) ? x[base + T * j] : none;
    if (r) {
      __half b[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) b[j] = in(j) ? r[base + T * j] : none;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        s[j] = __hadd_rn(b[j], s[j]);
        if (in(j)) sum[base + T * j] = s[j];
      }
    }
  };
  float ss = 0.0f, m = 0.0f;
  auto stat8 = [&](auto whole, int base, const __half (&s)[8]) {
    auto in = [&](int j) { return whole() || base + T * j < A.k; };
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float f = __half2float(s[j]);
      if (A.gamma) {
        ss = fmaf(f, f, ss);
        f *= in(j) ? __half2float(A.gamma[base + T * j]) : 0.0f;
      }
      m = max_abs(m, f, 0.0f);
    }
  };
  __half s[E][8];
#pragma unroll
  for (int i = 0; i < E; ++i) each(t + 8 * T * i, [&](auto w) { load8(w, t + 8 * T * i, s[i]); });
#pragma unroll
  for (int i = 0; i < E; ++i) each(t + 8 * T * i, [&](auto w) { stat8(w, t + 8 * T * i, s[i]); });
  for (int base = t + 8 * T * E; base < A.k; base += 8 * T) {
    __half v[8];
    load8(std::false_type{}, base, v);
    stat8(std::false_type{}, base, v);
  }
  const bool scaling = A.values || t < kWarp;
  uint32_t mbits;
  reduce_row<T, true>(ss, m, mbits, scaling);
  const float scale = scaling ? row_scale(A, ss, mbits) : 0.0f, inv = row_factor(mbits);
  if (t == 0) A.scales[row] = scale;
  const bool dead = mbits >= 0x7F800000u;
  int8_t* codes = A.codes + row * A.ldc;
  __half* values = A.values ? A.values + row * A.ldv : nullptr;
  auto give8 = [&](auto whole, int base, const __half (&s)[8]) {
    auto in = [&](int j) { return whole() || base + T * j < A.k; };
    float f[8], c[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      f[j] = __half2float(s[j]);
      if (A.gamma) f[j] *= in(j) ? __half2float(A.gamma[base + T * j]) : 0.0f;
      if (dead) f[j] = 0.0f;
    }
    row_codes(f, inv, mbits, c);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (in(j)) {
        codes[base + T * j] = static_cast<int8_t>(__float_as_uint(c[j]) & 0xFFu);
        if (values) values[base + T * j] = __float2half_rn((c[j] - kMagic) * scale);
      }
  };
#pragma unroll
  for (int i = 0; i < E; ++i) each(t + 8 * T * i, [&](auto w) { give8(w, t + 8 * T * i, s[i]); });
  const __half* again = r ? sum : x;
  for (int base = t + 8 * T * E; base < A.k; base += 8 * T) {
    __half v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = base + T * j < A.k ? again[base + T * j] : none;
    give8(std::false_type{}, base, v);
  }
}

template <int T>
static int launch(void (*kernel)(RowArgs), const RowArgs& A, cudaStream_t st) {
  constexpr int per = kCtaOf<T> / T;
  return lmps_launch_pdl(kernel, dim3((A.rows - 1) / per + 1), dim3(kCtaOf<T>), 0, st, A);
}

// `pieces` of eight elements, T threads a row.
template <int T, int E>
static int launch_pieces(const RowArgs& A, bool vec, cudaStream_t st) {
  if (!vec) return launch<T>(rows_any_kernel<T, E>, A, st);
  return launch<T>(A.gamma ? rows_vec_kernel<T, E, true> : rows_vec_kernel<T, E, false>, A, st);
}
template <int T>
static int launch_threads(const RowArgs& A, bool vec, int pieces, cudaStream_t st) {
  const int e = (pieces + T - 1) / T;
  if (e <= 1) return launch_pieces<T, 1>(A, vec, st);
  return e <= 2 ? launch_pieces<T, 2>(A, vec, st) : launch_pieces<T, 3>(A, vec, st);
}

// Four to nine pieces a thread (past six: neither gamma nor values).
template <int T>
static int launch_deep(const RowArgs& A, int pieces, cudaStream_t st) {
  if (pieces > 6 * T) return launch<T>(rows_vec_kernel<T, 9, false>, A, st);
  return launch<T>(A.gamma ? rows_vec_kernel<T, 6, true> : rows_vec_kernel<T, 6, false>, A, st);
}

// Threads a row (us at 16384 rows, else as said).  Where rows enough fill the SMs, as few as hold it in up to nine
// pieces each, so that the reduction is of fewer warps (8960 64 with 128, 72 with 256; 2048 17 with 32, 25 with 128);
// six with more to hold, gamma or the values (norm of 4096 48 with 128, 60 with 256), five with a residual (4096 72,
// 78; but 1536 33 with 32 threads, 31 with 64).  Of fewer rows as few threads as hold it in three pieces and make a
// quarter of what fits 148 SMs (with residual 600 x 1536: 3.4 with 128, 3.9 with 256; 2048 x 1536: 7.2 with 64, 8.0
// with 128); else a CTA, of 1024 for long rows up to one an SM (128 x 8960: 2.6, 2.8 with 256).
constexpr long long kFill = 148ll * 512, kFull = 148ll * 1536;
constexpr int kFewRows = 148;

static int launch_rows(const RowArgs& A, cudaStream_t st) {
  const bool vec = A.k % 8 == 0 && A.ldx % 8 == 0 && A.ldc % 8 == 0 && A.ldr % 8 == 0 && A.lds % 8 == 0 &&
                   A.ldv % 8 == 0 && lmps_aligned(A.x, 16) && lmps_aligned(A.residual, 16) &&
                   lmps_aligned(A.sum, 16) && lmps_aligned(A.gamma, 16) && lmps_aligned(A.codes, 8) &&
                   lmps_aligned(A.values, 16) && A.k <= kCta * 8 * 8;
  const int pieces = (A.k + 7) / 8;
  const int deep = A.residual ? 5 : A.gamma || A.values ? 6 : 9;
  auto fits = [&](int t, int most, long long fill) { return pieces <= most * t && A.rows * static_cast<long long>(t) >= fill; };
  if (vec && pieces > 3 * 32) {
    if (fits(32, deep, kFull)) return launch_deep<32>(A, pieces, st);
    if (fits(64, deep, kFull) && pieces > 3 * 64) return launch_deep<64>(A, pieces, st);
    if (fits(128, deep, kFull) && pieces > 3 * 128) return launch_deep<128>(A, pieces, st);
  }
  if (pieces <= 32 || fits(32, 3, kFill)) return launch_threads<32>(A, vec, pieces, st);
  if (pieces <= 64 || fits(64, 3, kFill)) return launch_threads<64>(A, vec, pieces, st);
  if (pieces <= 128 || fits(128, 3, kFill)) return launch_threads<128>(A, vec, pieces, st);
  if (pieces <= kCta || (pieces <= 3 * kCta && A.rows > kFewRows)) return launch_threads<kCta>(A, vec, pieces, st);
  if (pieces <= 1024 * 2 && A.rows <= kFewRows) return launch_pieces<1024, 2>(A, vec, st);
  if (!vec || pieces <= 5 * kCta) return launch_pieces<kCta, 5>(A, vec, st);
  return launch<kCta>(A.gamma ? rows_vec_kernel<kCta, 8, true> : rows_vec_kernel<kCta, 8, false>, A, st);
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
  if (k > q8::kMaxK) return LMPS_ERR_UNSUPPORTED;
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
  if (k > q8::kMaxK) return LMPS_ERR_UNSUPPORTED;
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
