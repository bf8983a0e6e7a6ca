// Shared by the attention kernels over the 4-bit KV cache: codes as fp16
// integers, the merge of split partials, argument checks.
#pragma once

#include "kv_q4.cuh"

namespace lmps {
namespace q4 {

constexpr int kMaxHeads = 8;  // query heads per KV head
constexpr float kScaleLog2 = kAttnScale * 1.4426950408889634f;  // scores in base 2

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t lop_or(uint32_t a, uint32_t mask) {  // (a & mask) | 0x64006400
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, 0x64006400, 0xEA;" : "=r"(d) : "r"(a), "r"(mask));
  return d;
}
// Codes (minus 8) of nibbles 0 and 4 (lo) or 1 and 5 (hi) of w as a half2:
// 0x6400 | n is 1024 + n, 0x6400 | n << 4 is 1024 + 16 n; both steps are exact.
__device__ __forceinline__ uint32_t codes_lo(uint32_t w) {
  const uint32_t x = lop_or(w, 0x000F000Fu);
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2(__ushort_as_half(0x6408), __ushort_as_half(0x6408)));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t codes_hi(uint32_t w) {
  const uint32_t x = lop_or(w, 0x00F000F0u);
  const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&x), __half2(__ushort_as_half(0x2C00), __ushort_as_half(0x2C00)),
                            __half2(__ushort_as_half(0xD480), __ushort_as_half(0xD480)));  // / 16 - 72
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Unnormalised results of the pieces of a call and where they lie.  Decode
// (rows_item 0): O [piece][n_q][128], row r has pieces[r].y of them from
// pieces[r].x on.  Many queries a sequence: O [piece][n_kv][rows_item][128] of
// blocks of rows_item (query, head) rows; entry (block from the last) * batch +
// sequence of `pieces`, and query i >= q_lens[b] is left alone (q_lens NULL:
// none is).  ml: per O row the max (base 2) and the sum.
struct Partials {
  float* o;
  float2* ml;
  const int2* pieces;
  __half* out;  // [rows, n_q * 128]
  int n_q, n_kv, rows_item;
  const int32_t* q_lens;
  int seq, batch, n_blocks;
};
// Launches the merge of `rows` rows.
int combine_launch(const Partials& p, int rows, cudaStream_t stream);
// LMPS_OK, or why the attention entry points refuse these sizes.
int check_attention(int n_pages, int max_pages, int page_size, int n_q_heads, int n_kv_heads, int head_dim,
                    int max_seq_len, int n_splits);

}  // namespace q4
}  // namespace lmps
