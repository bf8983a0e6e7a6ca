// RoPE on q and k of the fused q|k|v rows, then the append of the K and V rows
// to the paged 4-bit cache (kv_q4.cuh: format and quantiser).
//
// One CTA per token row: the row's 64 (cos, sin) pairs are computed once in
// fp64, then each warp takes whole heads (128 elements, 4 per lane).
#include "kv_q4.cuh"

namespace lmps {
namespace q4 {

constexpr int kAppendThreads = 256;

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
  int n_q, style;
};

__global__ void __launch_bounds__(kAppendThreads) rope_kv_append_q4_kernel(const AppendParams P) {
  lmps_pdl_trigger();
  lmps_pdl_wait();
  __shared__ double2 cs[kDim / 2];
  const int row = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int p = P.pos[row];
  if (p < 0) return;  // a row that is not in use
  if (p >= P.c.max_pages * P.c.page_size) {
    if (tid == 0) raise_error(P.c.error, kErrPosition);
    return;
  }
  const int pi = P.c.page_index(p), off = p - pi * P.c.page_size;
  const int page = P.c.bt[static_cast<size_t>(row) * P.c.max_pages + pi];
  if (page < 0 || page >= P.c.n_pages) {
    if (tid == 0) raise_error(P.c.error, kErrPage);
    return;
  }
  if (tid < kDim / 2) rope_cos_sin(p, P.inv_freq[tid], cs[tid].x, cs[tid].y);
  __syncthreads();
  const int n_kv = P.c.n_kv, heads = P.n_q + 2 * n_kv;
  const __half* src = P.qkv + static_cast<size_t>(row) * heads * kDim;
  for (int h = warp; h < heads; h += kAppendThreads / kWarp) {
    union {
      uint2 u;
      __half x[4];
    } e;
    e.u = *reinterpret_cast<const uint2*>(src + h * kDim + 4 * lane);
    const bool is_v = h >= P.n_q + n_kv;
    if (!is_v) rotate_head(e.x, cs, P.style, lane);
    if (h < P.n_q) {
      *reinterpret_cast<uint2*>(P.q_out + (static_cast<size_t>(row) * P.n_q + h) * kDim + 4 * lane) = e.u;
      continue;
    }
    const int kvh = h - P.n_q - (is_v ? n_kv : 0);
    const float x[4] = {__half2float(e.x[0]), __half2float(e.x[1]), __half2float(e.x[2]), __half2float(e.x[3])};
    float scale;
    const uint32_t w = quantise_row(x, scale);
    uint8_t* block = (is_v ? P.v_pool : P.k_pool) + P.c.block(page, kvh);
    *reinterpret_cast<uint16_t*>(block + off * kCodeBytes + 2 * lane) = static_cast<uint16_t>(w);
    if ((lane & 7) == 0)
      *reinterpret_cast<__half*>(block + P.c.page_size * kCodeBytes + off * 8 + (lane >> 3) * 2) = __float2half_rn(scale);
    __half* copy = is_v ? P.v_out : P.k_out;
    if (copy) {
#pragma unroll
      for (int i = 0; i < 4; ++i) e.x[i] = __float2half_rn(nib_code(w, i) * scale);
      *reinterpret_cast<uint2*>(copy + (static_cast<size_t>(row) * n_kv + kvh) * kDim + 4 * lane) = e.u;
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
  if (head_dim != q4::kDim || page_size % q4::kRun != 0) return LMPS_ERR_UNSUPPORTED;
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
  return lmps_launch_pdl(q4::rope_kv_append_q4_kernel, dim3(rows), dim3(q4::kAppendThreads), 0, lmps_stream(stream),
                         P);
}
