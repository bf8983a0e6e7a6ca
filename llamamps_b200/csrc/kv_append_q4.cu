// RoPE on q and k of the fused q|k|v rows, then the append of the K and V rows
// to the paged 4-bit cache (kv_q4.cuh: format and quantiser).
//
// A CTA takes one token row, or four of a long call (so that all threads have
// a cosine to compute): the rows' 64 (cos, sin) pairs once in fp64, q in units
// of 16 bytes a thread, then a warp per two K or V rows (8 elements a lane).
//
// One row is launch and latency (3.3 us, as are 64).  A prompt of 8 x 2048 rows
// (12 query, 2 KV heads: 139 MB) takes 29.9 us = 4.6 TB/s, 0.71 of the measured
// copy rate; its instructions are the rotations and the quantiser, whose
// maximum and scale a row's 16 lanes share (32 lanes of 4 elements: 33.0 us).
// K is rotated in fp64 so that the rounding to fp16, and with it every code, is
// that of the exact formula.
#include "kv_q4.cuh"

namespace lmps {
namespace q4 {

constexpr int kAppendThreads = 256;
constexpr int kSmallRows = 1024;  // up to here a CTA per token, then per 4

struct AppendParams {
  const __half* qkv;
  const int32_t* pos;
  const float* inv_freq;
  __half* q_out;
  __half* k_out;  // optional: the cached rows' values
  __half* v_out;
  uint8_t* k_pool;
  uint8_t* v_pool;
  Cache c;
  int n_q, style, rows;
};

// The pair in one word (interleaved), or two pairs with their second elements in another word (NeoX).
__device__ __forceinline__ void rotate_word(uint32_t& w, float2 c) {
  const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&w));
  float2 y;
  rope_rotate32(x.x, x.y, c, y.x, y.y);
  const __half2 h = __floats2half2_rn(y.x, y.y);
  w = *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void rotate_words(uint32_t& a, uint32_t& b, float2 c0, float2 c1) {
  const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&a));
  const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&b));
  float2 u, v;
  rope_rotate32(x.x, y.x, c0, u.x, v.x);
  rope_rotate32(x.y, y.y, c1, u.y, v.y);
  const __half2 hu = __floats2half2_rn(u.x, u.y), hv = __floats2half2_rn(v.x, v.y);
  a = *reinterpret_cast<const uint32_t*>(&hu);
  b = *reinterpret_cast<const uint32_t*>(&hv);
}

template <int kTokens, int kStyle>
__global__ void __launch_bounds__(kAppendThreads) rope_kv_append_q4_kernel(const AppendParams P) {
  lmps_pdl_trigger();
  lmps_pdl_wait();
  __shared__ double2 csd[kTokens][kDim / 2];                // K's rotation
  __shared__ __align__(16) float2 csf[kTokens][kDim / 2];  // q's
  constexpr int kPer = kAppendThreads / kTokens;           // threads of a token
  constexpr int kUnit = kStyle == LMPS_ROPE_INTERLEAVED ? 8 : 16;  // elements a thread rotates at a time
  constexpr int kAhead = kUnit == 8 ? 4 : 2;                       // units loaded before the table is ready
  const int tid = threadIdx.x, lane = tid & 31, t = tid / kPer, l = tid % kPer;
  const int row = blockIdx.x * kTokens + t;
  const int n_kv = P.c.n_kv, heads = P.n_q + 2 * n_kv, units = P.n_q * (kDim / kUnit);
  const bool used = row < P.rows;
  const __half* src = P.qkv + static_cast<size_t>(used ? row : 0) * heads * kDim;
  // first element of unit u (NeoX: of its first halves; the second are 64 on)
  auto at = [](int u) { return kUnit == 8 ? 8 * u : (u >> 3) * kDim + 8 * (u & 7); };
  // everything that does not wait for the position: q units, and the first K or V row of this warp
  uint4 a[kAhead], b[kAhead];
#pragma unroll
  for (int k = 0; k < kAhead; ++k) {
    const int u = l + k * kPer;
    if (u < units) {
      a[k] = *reinterpret_cast<const uint4*>(src + at(u));
      if (kUnit == 16) b[k] = *reinterpret_cast<const uint4*>(src + at(u) + kDim / 2);
    }
  }
  const int sub = lane >> 4, l16 = lane & 15, r0 = 2 * (l >> 5);  // K and V: 16 lanes a row, 8 elements a lane
  uint4 kv = make_uint4(0u, 0u, 0u, 0u);
  if (r0 < 2 * n_kv) kv = *reinterpret_cast<const uint4*>(src + (P.n_q + r0 + sub) * kDim + 8 * l16);

  const int p = used ? P.pos[row] : -1;
  int page = -1, off = 0;
  if (p >= P.c.max_pages * P.c.page_size) {
    if (l == 0) raise_error(P.c.error, kErrPosition);
  } else if (p >= 0) {
    const int pi = P.c.page_index(p);
    off = p - pi * P.c.page_size;
    page = P.c.bt[static_cast<size_t>(row) * P.c.max_pages + pi];
    if (page < 0 || page >= P.c.n_pages) {
      if (l == 0) raise_error(P.c.error, kErrPage);
      page = -1;
    }
  }
  if (l < kDim / 2) {
    double2 d;
    rope_cos_sin(p, P.inv_freq[l], d.x, d.y);
    csd[t][l] = d;
    csf[t][l] = make_float2(static_cast<float>(d.x), static_cast<float>(d.y));
  }
  __syncthreads();
  if (page < 0) return;  // (uniform in a warp; no barrier follows) the row is left alone
  __half* q_out = P.q_out + static_cast<size_t>(row) * P.n_q * kDim;
  auto rotate = [&](int u, uint4 x, uint4 y) {
    const float4* cs = reinterpret_cast<const float4*>(&csf[t][kUnit == 8 ? 4 * (u & 15) : 8 * (u & 7)]);
    uint32_t* px = &x.x;
    uint32_t* py = &y.x;
#pragma unroll
    for (int e = 0; e < 4; e += kUnit == 8 ? 2 : 1) {
      const float4 c = cs[kUnit == 8 ? e / 2 : e];
      if (kUnit == 8) {
        rotate_word(px[e], make_float2(c.x, c.y));
        rotate_word(px[e + 1], make_float2(c.z, c.w));
      } else {
        rotate_words(px[e], py[e], make_float2(c.x, c.y), make_float2(c.z, c.w));
      }
    }
    *reinterpret_cast<uint4*>(q_out + at(u)) = x;
    if (kUnit == 16) *reinterpret_cast<uint4*>(q_out + at(u) + kDim / 2) = y;
  };
#pragma unroll
  for (int k = 0; k < kAhead; ++k)
    if (l + k * kPer < units) rotate(l + k * kPer, a[k], b[k]);
  for (int u = l + kAhead * kPer; u < units; u += kPer) {
    const uint4 x = *reinterpret_cast<const uint4*>(src + at(u));
    rotate(u, x, kUnit == 16 ? *reinterpret_cast<const uint4*>(src + at(u) + kDim / 2) : x);
  }
  // K and V (their 2 n_kv rows): a warp per two rows of 128, the next rows' load ahead
  constexpr int kStride = 2 * (kPer / kWarp);
  for (int r = r0; r < 2 * n_kv; r += kStride) {
    union {
      uint4 u;
      __half x[8];
    } e, rot;
    e.u = kv;
    if (r + kStride < 2 * n_kv)
      kv = *reinterpret_cast<const uint4*>(src + (P.n_q + r + kStride + sub) * kDim + 8 * l16);
    const bool is_v = r + sub >= n_kv;
    const int kvh = r + sub - (is_v ? n_kv : 0);
    if (r < n_kv) {  // (uniform) one K row at least
      rot.u = e.u;
      rotate_head(rot.x, csd[t], kStyle, lane);
      if (!is_v) e.u = rot.u;
    }
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __half2float(e.x[i]);
    float scale;
    const uint32_t w = quantise_row(x, scale);
    uint8_t* block = (is_v ? P.v_pool : P.k_pool) + P.c.block(page, kvh);
    *reinterpret_cast<uint32_t*>(block + off * kCodeBytes + 4 * l16) = w;
    if ((lane & 3) == 0)
      *reinterpret_cast<__half*>(block + P.c.page_size * kCodeBytes + off * 8 + (l16 >> 2) * 2) = __float2half_rn(scale);
    __half* copy = is_v ? P.v_out : P.k_out;
    if (copy) {
#pragma unroll
      for (int i = 0; i < 8; ++i) e.x[i] = __float2half_rn(nib_code(w, i) * scale);
      *reinterpret_cast<uint4*>(copy + (static_cast<size_t>(row) * n_kv + kvh) * kDim + 8 * l16) = e.u;
    }
  }
}

}  // namespace q4
}  // namespace lmps

using namespace lmps;

extern "C" int lmps_rope_kv_append_q4(const uint16_t* qkv, const int32_t* pos, const float* inv_freq,
                                      uint16_t* q_out, uint16_t* k_out, uint16_t* v_out, uint8_t* k_pool,
                                      uint8_t* v_pool, int n_pages, const int32_t* block_table, int max_pages,
                                      int page_size, int n_q_heads, int n_kv_heads, int head_dim, int rows,
                                      int style, int32_t* error, void* stream) {
  LMPS_CHECK_ARG(qkv && pos && inv_freq && q_out && k_pool && v_pool && block_table);
  LMPS_CHECK_ARG(rows >= 1 && n_pages >= 1 && max_pages >= 1 && page_size >= 1 && n_q_heads >= 1 && n_kv_heads >= 1);
  LMPS_CHECK_ARG(static_cast<long long>(max_pages) * page_size <= 1LL << 29);
  LMPS_CHECK_ARG(style == LMPS_ROPE_INTERLEAVED || style == LMPS_ROPE_NEOX);
  if (head_dim != q4::kDim || page_size % q4::kRun != 0 || page_size > q4::kMaxPage) return LMPS_ERR_UNSUPPORTED;
  LMPS_CHECK_ARG(lmps_aligned(qkv, 16) && lmps_aligned(q_out, 16) && lmps_aligned(k_out, 16) &&
                 lmps_aligned(v_out, 16) && lmps_aligned(k_pool, 16) && lmps_aligned(v_pool, 16));
  q4::AppendParams P{};
  P.qkv = reinterpret_cast<const __half*>(qkv);
  P.pos = pos;
  P.inv_freq = inv_freq;
  P.q_out = reinterpret_cast<__half*>(q_out);
  P.k_out = reinterpret_cast<__half*>(k_out);
  P.v_out = reinterpret_cast<__half*>(v_out);
  P.k_pool = k_pool;
  P.v_pool = v_pool;
  P.c = q4::Cache{k_pool, v_pool, block_table, n_pages, max_pages, page_size, n_kv_heads,
                  q4::page_shift_of(page_size), error};
  P.n_q = n_q_heads;
  P.style = style;
  P.rows = rows;
  // a CTA per token while that does not fill the GPU, else four tokens a CTA
  const bool il = style == LMPS_ROPE_INTERLEAVED, few = rows <= q4::kSmallRows;
  const auto kernel = il ? (few ? q4::rope_kv_append_q4_kernel<1, LMPS_ROPE_INTERLEAVED>
                                : q4::rope_kv_append_q4_kernel<4, LMPS_ROPE_INTERLEAVED>)
                         : (few ? q4::rope_kv_append_q4_kernel<1, LMPS_ROPE_NEOX>
                                : q4::rope_kv_append_q4_kernel<4, LMPS_ROPE_NEOX>);
  return lmps_launch_pdl(kernel, dim3(few ? rows : (rows + 3) / 4), dim3(q4::kAppendThreads), 0, lmps_stream(stream),
                         P);
}
